// Root-mean-square norm of a residual's sum, and dropout whose mask is never
// stored.
//
//   s = residual + drop(x),  rstd_n = 1 / sqrt(mean_f s_nf^2 + eps),
//   y_nf = s_nf rstd_n gamma_f
// backward, n_nf = s_nf rstd_n, d_nf = gamma_f dy_nf:
//   ds = dsum + rstd (d - n mean_f(d n)),  dresidual = ds, dx = drop(ds),
//   dgamma_f (+)= sum_n dy_nf n_nf
//
// Matrices are ColMajor [N, F]: the features of a row lie N apart.  Up to 1024 features
// (back, of less than 6000 rows, up to 512) a block holds 32 rows, a line of every column,
// in registers and reads everything once.
// Of longer rows it would hold a part of a line of every column, each on a page of its
// own (4097 x 4099, forward, 203 us in blocks of 16 rows for 81 here), so a larger matrix
// goes through in tiles of 256 rows x 32 columns and more, a KiB in a row of every
// column, twice: the first launch leaves each tile's sums over its columns, the second
// joins them and reads s (and dy) again, for the most part from the caches.  Where a few
// rows are all there is, one block does it.  The sums over a row are kept in 64 bits,
// which neither overflow nor vanish for any finite fp32 row.
//
// Bound by memory: 8192 x 512 with dropout takes 14.4 us forward (67 MB, 4.7 TB/s) and 18.0
// back (84 MB, 4.7 TB/s), a round of one block a CU, which loads, adds up and then stores,
// and 3.8 for dgamma; 8192 x 1024 without 23.5 and 24.3; 4097 x 4099 in tiles 48 + 29 us
// forward (375 MB, 4.9 TB/s) and 30 + 57 back (462 MB, 5.3 TB/s), of which reading s and dy
// again is a fifth and a third.  Dropout alone: 8192 x 2048 20.6 us, 6.5 TB/s with its
// input in the caches (24 among other work).
//
// Element j of the [N, F] storage is kept where the generator's word for
// position + j says so; the backward draws the same words again.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "common.hpp"
#include "dropout_rng.hpp"

namespace cnhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Drop {
  uint32_t limit;  // 2^24: everything is kept
  float scale;
  uint64_t seed, offset;
  const uint64_t* counter;
};
__device__ __forceinline__ uint64_t first_word(const Drop& d) {
  return d.seed + (d.offset + (d.counter ? *d.counter : 0)) * kDropoutStep;
}
__device__ __forceinline__ float dropped(const Drop& d, uint64_t word, float x) {
  return dropout_top24(word) < d.limit ? x * d.scale : 0.f;
}

// ---------------------------------------------------------------- dropout
__global__ void __launch_bounds__(256) dropout_seeded_kernel(const float* x, float* y, int64_t n, Drop d) {
  const int64_t stride = (int64_t)gridDim.x * 256 * 4;
  const uint64_t z0 = first_word(d);
  for (int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; j < n; j += stride) {
    const uint64_t z = z0 + (uint64_t)j * kDropoutStep;
    if (j + 4 <= n) {
      f32x4 v = *reinterpret_cast<const f32x4u*>(x + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = dropped(d, z + (uint64_t)e * kDropoutStep, v[e]);
      *reinterpret_cast<f32x4u*>(y + j) = v;
    } else {
      for (int e = 0; j + e < n; ++e) y[j + e] = dropped(d, z + (uint64_t)e * kDropoutStep, x[j + e]);
    }
  }
}

__global__ void dropout_advance_kernel(uint64_t* counter, uint64_t n) { *counter += n; }

// ------------------------------------------------------------------- norm
struct NormArgs {
  const float *x, *residual, *gamma;
  float *y, *sum, *rstd;
  const float *s, *dy, *dsum;
  float *dx, *dresidual, *dgamma;
  int64_t N, F;
  double eps, inv_f;
  Drop drop;
  int accumulate;
  int shift;          // few rows: log2 of the rows of a block; tiles: of the lanes along the rows
  int row_tiles, col_tiles;
  int chunks;         // times that a block of a tile goes through K columns a thread
  double* part;       // [col_tiles][N]: sums over a tile's columns
  float* gamma_part;  // [row_tiles][F]: sums over a tile's rows
};

constexpr int kNormThreads = 1024, kNormWaves = kNormThreads / 64;
constexpr int kTileThreads = 512, kTileWaves = kTileThreads / 64;

// 1 / sqrt(v) to fp32's precision and range.
__device__ __forceinline__ float inv_sqrt(double v) {
  double r = __builtin_amdgcn_rsq(v);
  r = r * fma(-0.5 * v * r, r, 1.5);
  return (float)r;
}

// ---- few rows
// Where a thread's elements lie: feature `first` + k cols of its row for k = 0, 1, ...,
// at[j] of a matrix's part(k).  What the lanes of a wave share is kept apart, so that an
// element costs one 32-bit address and not one of 64 bits in every matrix.
struct Seat {
  int rows, cols, r;
  int64_t step, base, first0;  // features and elements before the wave's first
  uint32_t lane_f, j;          // and the lane's own
  __device__ __forceinline__ Seat(int64_t N, int shift) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    rows = 1 << shift;
    cols = kNormThreads >> shift;
    r = lane & (rows - 1);
    lane_f = lane >> shift;
    first0 = (int64_t)wave * (64 >> shift);
    base = N * first0;
    step = N * cols;
    j = (uint32_t)r + (uint32_t)N * lane_f;
  }
  __device__ __forceinline__ int64_t part(int k) const { return base + k * step; }
  __device__ __forceinline__ bool has(int k, int64_t F) const { return first0 + (int64_t)k * cols + lane_f < F; }
};

// The sum over a block's threads with the same row (thread % rows), in every one of them.
__device__ __forceinline__ double row_sum(double v, int shift, double (*part)[64]) {
  const int rows = 1 << shift, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = rows; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  if (lane < rows) part[wave][lane] = v;
  __syncthreads();
  double t = 0.0;
  const int r = lane & (rows - 1);
#pragma unroll
  for (int w = 0; w < kNormWaves; ++w) t += part[w][r];
  return t;
}

// K: a thread's features at most.
template <int K, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_few_fwd_kernel(NormArgs a) {
#pragma clang fp contract(off)
  __shared__ double part[kNormWaves][64];
  const Seat w(a.N, a.shift);
  const int64_t n0 = (int64_t)blockIdx.x << a.shift;
  const bool in = n0 + w.r < a.N;
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)w.j * kDropoutStep : 0;
  float s[K];
  double q = 0.0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    s[k] = 0.f;
    if (!in || !w.has(k, a.F)) continue;
    const int64_t o = n0 + w.part(k);
    float v = (a.x + o)[w.j];
    if (DROP) v = dropped(a.drop, z0 + (uint64_t)o * kDropoutStep, v);
    s[k] = a.residual ? (a.residual + o)[w.j] + v : v;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    q = fma((double)s[k], (double)s[k], q);
    if (a.sum && in && w.has(k, a.F)) (a.sum + n0 + w.part(k))[w.j] = s[k];
  }
  const float rstd = inv_sqrt(row_sum(q, a.shift, part) * a.inv_f + a.eps);
  if (!in) return;
  if (a.rstd && threadIdx.x < (unsigned)w.rows) a.rstd[n0 + w.r] = rstd;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (w.has(k, a.F)) (a.y + n0 + w.part(k))[w.j] = (s[k] * rstd) * (a.gamma + w.first0 + (int64_t)k * w.cols)[w.lane_f];
}

template <int K, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_few_bwd_kernel(NormArgs a) {
  __shared__ double part[kNormWaves][64];
  const Seat w(a.N, a.shift);
  const int64_t n0 = (int64_t)blockIdx.x << a.shift;
  const bool in = n0 + w.r < a.N;
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)w.j * kDropoutStep : 0;
  const float rstd = in ? a.rstd[n0 + w.r] : 0.f;
  float u[K], d[K];  // the normed row, and the gradient at it
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool on = in && w.has(k, a.F);
    const int64_t o = n0 + w.part(k);
    u[k] = on ? (a.s + o)[w.j] * rstd : 0.f;
    d[k] = on ? (a.dy + o)[w.j] : 0.f;
  }
  double q = 0.0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    // dgamma's part: over the rows of the block, lanes side by side
    float dg = d[k] * u[k];
    for (int o = w.rows >> 1; o > 0; o >>= 1) dg += __shfl_xor(dg, o, 64);
    if (w.has(k, a.F)) {
      const int64_t f = w.first0 + (int64_t)k * w.cols;
      if (w.r == 0) (a.gamma_part + blockIdx.x * a.F + f)[w.lane_f] = dg;
      d[k] *= (a.gamma + f)[w.lane_f];
    }
    q = fma((double)d[k], (double)u[k], q);
  }
  const float c = (float)(row_sum(q, a.shift, part) * a.inv_f);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!in || !w.has(k, a.F)) continue;
    const int64_t o = n0 + w.part(k);
    float g = rstd * fmaf(-u[k], c, d[k]);
    if (a.dsum) g += (a.dsum + o)[w.j];
    if (a.dresidual) (a.dresidual + o)[w.j] = g;
    (a.dx + o)[w.j] = DROP ? dropped(a.drop, z0 + (uint64_t)o * kDropoutStep, g) : g;
  }
}

// dgamma (+)= the tiles' parts, in order: 64 features a block, its waves share the parts.
__device__ __forceinline__ void join_gamma(const NormArgs& a, int64_t block, float (*sum)[64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f = block * 64 + lane;
  float t = 0.f;
  if (f < a.F) {
#pragma unroll 8
    for (int b = wave; b < a.row_tiles; b += kTileWaves) t += a.gamma_part[(int64_t)b * a.F + f];
  }
  sum[wave][lane] = t;
  __syncthreads();
  if (wave || f >= a.F) return;
  for (int w = 1; w < kTileWaves; ++w) t += sum[w][lane];
  a.dgamma[f] = a.accumulate ? a.dgamma[f] + t : t;
}
// The same in a launch of its own, 16 features a block.
__global__ void __launch_bounds__(kNormThreads) rms_norm_gamma_kernel(NormArgs a) {
  __shared__ float sum[kNormWaves][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f = (int64_t)blockIdx.x * 16 + (lane & 15);
  float t = 0.f;
  if (f < a.F) {
#pragma unroll 4
    for (int b = threadIdx.x >> 4; b < a.row_tiles; b += kNormThreads / 16) t += a.gamma_part[(int64_t)b * a.F + f];
  }
  t += __shfl_xor(t, 16, 64);
  t += __shfl_xor(t, 32, 64);
  if (lane < 16) sum[wave][lane] = t;
  __syncthreads();
  if (threadIdx.x >= 16 || f >= a.F) return;
  t = 0.f;
#pragma unroll
  for (int w = 0; w < kNormWaves; ++w) t += sum[w][lane];
  a.dgamma[f] = a.accumulate ? a.dgamma[f] + t : t;
}

// ---- tiles
constexpr int K = 4;  // a thread's columns at a time
// 2^shift lanes along the rows, 4 rows each, and chunks times K times (kTileThreads >>
// shift) columns; what stays in registers is a chunk's.
// Row tiles lie side by side in the order of the blocks.  WHOLE: all of the tile's rows
// and columns exist, and every thread's loads go out one after the other (behind the
// tests of a ragged tile each would be waited for).
template <bool WHOLE>
struct TileSeat {
  int64_t n, f0, base;  // the lane's first row; the wave's first column, its first element
  int64_t step;
  uint32_t lane_f, j;
  int cols, row, tile_r, tile_c, left;  // rows of this lane's 4 that exist
  __device__ __forceinline__ TileSeat(const NormArgs& a, int bid) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    tile_r = bid % a.row_tiles;
    tile_c = bid / a.row_tiles;
    cols = kTileThreads >> a.shift;
    row = 4 * (lane & ((1 << a.shift) - 1));
    lane_f = lane >> a.shift;
    const int64_t n0 = (int64_t)tile_r << (a.shift + 2);
    f0 = (int64_t)tile_c * a.chunks * (K * cols) + (int64_t)wave * (64 >> a.shift);
    n = n0 + row;
    base = n0 + a.N * f0;
    step = a.N * cols;
    j = (uint32_t)row + (uint32_t)a.N * lane_f;
    left = WHOLE || n + 4 <= a.N ? 4 : n < a.N ? (int)(a.N - n) : 0;
  }
  __device__ __forceinline__ bool has(int k, int64_t F) const { return WHOLE || f0 + (int64_t)k * cols + lane_f < F; }
  __device__ __forceinline__ int64_t at(int k) const { return base + k * step; }
  __device__ __forceinline__ f32x4 get(const float* p, int k, int64_t F) const {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (!has(k, F)) return v;
    const float* q = p + at(k) + j;
    if (WHOLE || left == 4) return f32x4(*reinterpret_cast<const f32x4u*>(q));
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) v[e] = q[e];
    return v;
  }
  __device__ __forceinline__ void put(float* p, int k, int64_t F, const f32x4& v) const {
    if (!has(k, F)) return;
    float* q = p + at(k) + j;
    if (WHOLE || left == 4) {
      *reinterpret_cast<f32x4u*>(q) = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) q[e] = v[e];
  }
  __device__ __forceinline__ float of_column(const float* p, int k, int64_t F) const {
    return has(k, F) ? (p + f0 + (int64_t)k * cols)[lane_f] : 0.f;
  }
  // dropout of the lane's 4 elements in column k; z0: the word of the lane's own offset
  __device__ __forceinline__ f32x4 drop(const Drop& d, uint64_t z0, int k, f32x4 v) const {
    const uint64_t z = z0 + (uint64_t)at(k) * kDropoutStep;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = dropped(d, z + (uint64_t)e * kDropoutStep, v[e]);
    return v;
  }
};

// The tile's sums over its columns -> part; q: of the thread's rows.
template <class Seat_>
__device__ __forceinline__ void leave_sums(const NormArgs& a, const Seat_& t, double (&q)[4], double (*lds)[256]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lanes = 1 << a.shift;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    for (int o = lanes; o < 64; o <<= 1) q[e] += __shfl_xor(q[e], o, 64);
    if (lane < lanes) lds[wave][4 * lane + e] = q[e];
  }
  __syncthreads();
  const int r = threadIdx.x;
  const int64_t n = ((int64_t)t.tile_r << (a.shift + 2)) + r;
  if (r >= 4 * lanes || n >= a.N) return;
  double v = 0.0;
#pragma unroll
  for (int w = 0; w < kTileWaves; ++w) v += lds[w][r];
  a.part[(int64_t)t.tile_c * a.N + n] = v;
}
// The sums over all columns of the thread's 4 rows; the threads share them out.
template <class Seat_>
__device__ __forceinline__ void all_sums(const NormArgs& a, const Seat_& t, double (&q)[4], double (*lds)[256]) {
  const int rows = 4 << a.shift, r = threadIdx.x & (rows - 1), g = threadIdx.x >> (a.shift + 2),
            groups = kTileThreads >> (a.shift + 2);
  const int64_t n = ((int64_t)t.tile_r << (a.shift + 2)) + r;
  double v = 0.0;
  if (n < a.N) {
#pragma unroll 4
    for (int c = g; c < a.col_tiles; c += groups) v += a.part[(int64_t)c * a.N + n];
  }
  // groups of fewer rows than a line of lds share one: [groups rows / 256][256]
  (&lds[0][0])[threadIdx.x] = v;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = 0.0;
    for (int k = 0; k < min(groups, a.col_tiles); ++k) q[e] += (&lds[0][0])[k * rows + t.row + e];
  }
}

__device__ __forceinline__ bool whole_tile(const NormArgs& a, int bid) {
  const int64_t rows = (int64_t)4 << a.shift, cols = (int64_t)a.chunks * K * (kTileThreads >> a.shift);
  return (bid % a.row_tiles + 1) * rows <= a.N && (bid / a.row_tiles + 1) * cols <= a.F;
}

template <bool DROP, bool WHOLE>
__device__ __forceinline__ void rms_norm_sum_tile(const NormArgs& a, double (*lds)[256]) {
#pragma clang fp contract(off)
  const TileSeat<WHOLE> t(a, (int)blockIdx.x);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)t.j * kDropoutStep : 0;
  double q[4] = {};
  for (int k0 = 0; k0 < a.chunks * K; k0 += K) {
    f32x4 s[K], r[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      s[k] = t.get(a.x, k0 + k, a.F);
      if (a.residual) r[k] = t.get(a.residual, k0 + k, a.F);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (DROP) s[k] = t.drop(a.drop, z0, k0 + k, s[k]);
      if (a.residual) s[k] = r[k] + s[k];
      if (a.sum) t.put(a.sum, k0 + k, a.F, s[k]);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = fma((double)s[k][e], (double)s[k][e], q[e]);
    }
  }
  leave_sums(a, t, q, lds);
}
template <bool DROP>
__global__ void __launch_bounds__(kTileThreads) rms_norm_sum_kernel(NormArgs a) {
  __shared__ double lds[kTileWaves][256];
  if (whole_tile(a, (int)blockIdx.x)) rms_norm_sum_tile<DROP, true>(a, lds);
  else rms_norm_sum_tile<DROP, false>(a, lds);
}

template <bool DROP, bool WHOLE>
__device__ __forceinline__ void rms_norm_apply_tile(const NormArgs& a, double (*lds)[256]) {
#pragma clang fp contract(off)
  const TileSeat<WHOLE> t(a, (int)blockIdx.x);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)t.j * kDropoutStep : 0;
  f32x4 s[K];
  auto get = [&](int k0) {
    if (a.sum) {
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] = t.get(a.sum, k0 + k, a.F);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        s[k] = t.get(a.x, k0 + k, a.F);
        if (DROP) s[k] = t.drop(a.drop, z0, k0 + k, s[k]);
        if (a.residual) s[k] = t.get(a.residual, k0 + k, a.F) + s[k];
      }
    }
  };
  get(0);
  double q[4];
  all_sums(a, t, q, lds);
  f32x4 rstd;
#pragma unroll
  for (int e = 0; e < 4; ++e) rstd[e] = inv_sqrt(q[e] * a.inv_f + a.eps);
  if (a.rstd && t.tile_c == 0 && threadIdx.x < (1u << a.shift)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < t.left) a.rstd[t.n + e] = rstd[e];
  }
  for (int k0 = 0;;) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float g = t.of_column(a.gamma, k0 + k, a.F);
      t.put(a.y, k0 + k, a.F, (s[k] * rstd) * g);
    }
    k0 += K;
    if (k0 >= a.chunks * K) break;
    get(k0);
  }
}
template <bool DROP>
__global__ void __launch_bounds__(kTileThreads) rms_norm_apply_kernel(NormArgs a) {
  __shared__ double lds[kTileThreads / 256][256];
  if (whole_tile(a, (int)blockIdx.x)) rms_norm_apply_tile<DROP, true>(a, lds);
  else rms_norm_apply_tile<DROP, false>(a, lds);
}

// First of the backward: the sums of d n over a tile's columns and of dy n over its rows.
template <bool WHOLE>
__device__ __forceinline__ void rms_norm_dots_tile(const NormArgs& a, double (*lds)[256]) {
  const TileSeat<WHOLE> t(a, (int)blockIdx.x);
  f32x4 rstd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < t.left) rstd[e] = a.rstd[t.n + e];
  double q[4] = {};
  for (int k0 = 0; k0 < a.chunks * K; k0 += K) {
    f32x4 u[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      u[k] = t.get(a.s, k0 + k, a.F);
      d[k] = t.get(a.dy, k0 + k, a.F);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float g = t.of_column(a.gamma, k0 + k, a.F);
      float dg = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float n = u[k][e] * rstd[e];
        if (e < t.left) dg = fmaf(d[k][e], n, dg);
        q[e] = fma((double)(d[k][e] * g), (double)n, q[e]);
      }
      for (int o = (1 << a.shift) >> 1; o > 0; o >>= 1) dg += __shfl_xor(dg, o, 64);
      if (t.row == 0 && t.has(k0 + k, a.F))
        (a.gamma_part + (int64_t)t.tile_r * a.F + t.f0 + (int64_t)(k0 + k) * t.cols)[t.lane_f] = dg;
    }
  }
  leave_sums(a, t, q, lds);
}
__global__ void __launch_bounds__(kTileThreads) rms_norm_dots_kernel(NormArgs a) {
  __shared__ double lds[kTileWaves][256];
  if (whole_tile(a, (int)blockIdx.x)) rms_norm_dots_tile<true>(a, lds);
  else rms_norm_dots_tile<false>(a, lds);
}

// Second: dx and dresidual; the blocks behind the tiles join dgamma.
template <bool DROP, bool WHOLE>
__device__ __forceinline__ void rms_norm_grad_tile(const NormArgs& a, double (*lds)[256]) {
  const TileSeat<WHOLE> t(a, (int)blockIdx.x);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)t.j * kDropoutStep : 0;
  f32x4 u[K], d[K], p[K], rstd = {0.f, 0.f, 0.f, 0.f};
  auto get = [&](int k0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      u[k] = t.get(a.s, k0 + k, a.F);
      d[k] = t.get(a.dy, k0 + k, a.F);
      if (a.dsum) p[k] = t.get(a.dsum, k0 + k, a.F);
    }
  };
  get(0);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < t.left) rstd[e] = a.rstd[t.n + e];
  double q[4];
  all_sums(a, t, q, lds);
  float c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = (float)(q[e] * a.inv_f);
  for (int k0 = 0;;) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float gamma = t.of_column(a.gamma, k0 + k, a.F);
      f32x4 g;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = rstd[e] * fmaf(-(u[k][e] * rstd[e]), c[e], d[k][e] * gamma);
        if (a.dsum) g[e] += p[k][e];
      }
      if (a.dresidual) t.put(a.dresidual, k0 + k, a.F, g);
      t.put(a.dx, k0 + k, a.F, DROP ? t.drop(a.drop, z0, k0 + k, g) : g);
    }
    k0 += K;
    if (k0 >= a.chunks * K) break;
    get(k0);
  }
}
template <bool DROP>
__global__ void __launch_bounds__(kTileThreads) rms_norm_grad_kernel(NormArgs a) {
  __shared__ double lds[kTileThreads / 256][256];
  const int tiles = a.row_tiles * a.col_tiles;
  if ((int)blockIdx.x >= tiles) {
    join_gamma(a, (int)blockIdx.x - tiles, reinterpret_cast<float(*)[64]>(&lds[0][0]));
    return;
  }
  if (whole_tile(a, (int)blockIdx.x)) rms_norm_grad_tile<DROP, true>(a, lds);
  else rms_norm_grad_tile<DROP, false>(a, lds);
}

// ---- rows held
// Up to kHeldFeatures features: a block holds 32 rows, a line of every column, with all
// of their features in registers, and one launch does it (back, but for joining the blocks'
// parts of dgamma).  8 lanes go along the rows, 4
// rows each, and CH times kNormWaves kCols features, of which a wave has kCols side by
// side.  Behind the last feature a wave reads the last kCols again and counts and writes
// those that no other has (a test around its loads takes registers that there are not:
// 8192 x 1024, back, 77 us for 24).
constexpr int kHeldRows = 32;
// The blocks of an XCD (every eighth) take row tiles side by side: of an odd number of rows
// neighbours share lines.
__device__ __forceinline__ int held_tile(const NormArgs& a) {
  const int b = (int)blockIdx.x, n = a.row_tiles, x = b % 8;
  return x * (n / 8) + min(x, n % 8) + b / 8;
}

template <bool WHOLE>
struct HeldSeat {
  static constexpr int kCols = 256 / kHeldRows;  // of a wave, side by side
  int64_t n0, F, N;          // the block's first row
  int tile, row, left, f0;   // the lane's first of its rows, how many of them exist; the wave's first feature
  uint32_t lane_f, j;
  __device__ __forceinline__ HeldSeat(const NormArgs& a, int bid) : F(a.F), N(a.N), tile(bid) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    row = 4 * (lane & (kHeldRows / 4 - 1));
    lane_f = lane / (kHeldRows / 4);
    f0 = kCols * wave;
    n0 = (int64_t)bid * kHeldRows;
    j = (uint32_t)row + (uint32_t)a.N * lane_f;
    left = WHOLE || n0 + row + 4 <= N ? 4 : n0 + row < N ? (int)(N - n0 - row) : 0;
  }
  // The first of the wave's features: where they would end behind the last, those before.
  __device__ __forceinline__ int column(int k) const { return min(first(k), (int)F - kCols); }
  __device__ __forceinline__ int first(int k) const { return f0 + k * (kNormWaves * kCols); }
  __device__ __forceinline__ bool has(int k) const { return column(k) + (int)lane_f >= first(k); }
  __device__ __forceinline__ int64_t at(int k) const { return n0 + N * column(k); }
  __device__ __forceinline__ f32x4 get(const float* p, int k) const {
    const float* q = p + at(k) + j;
    if (WHOLE || left == 4) return f32x4(*reinterpret_cast<const f32x4u*>(q));
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) v[e] = q[e];
    return v;
  }
  __device__ __forceinline__ void put(float* p, int k, const f32x4& v) const {
    if (!has(k)) return;
    float* q = p + at(k) + j;
    if (WHOLE || left == 4) {
      *reinterpret_cast<f32x4u*>(q) = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) q[e] = v[e];
  }
  __device__ __forceinline__ float of_column(const float* p, int k) const { return (p + column(k))[lane_f]; }
  __device__ __forceinline__ f32x4 drop(const Drop& d, uint64_t z0, int k, f32x4 v) const {
    const uint64_t z = z0 + (uint64_t)at(k) * kDropoutStep;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = dropped(d, z + (uint64_t)e * kDropoutStep, v[e]);
    return v;
  }
};

// The sums over the block's features of the thread's 4 rows.
__device__ __forceinline__ void held_sums(double (&q)[4], int row, double (*part)[kHeldRows], double* sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    for (int o = kHeldRows / 4; o < 64; o <<= 1) q[e] += __shfl_xor(q[e], o, 64);
    if (lane < kHeldRows / 4) part[wave][row + e] = q[e];
  }
  __syncthreads();
  if (threadIdx.x < kHeldRows) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < kNormWaves; ++w) v += part[w][threadIdx.x];
    sum[threadIdx.x] = v;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = sum[row + e];
}

template <int CH, bool DROP, bool WHOLE>
__device__ __forceinline__ void rms_norm_held_fwd_tile(const NormArgs& a, int bid, double (*part)[kHeldRows], double* sum) {
#pragma clang fp contract(off)
  const HeldSeat<WHOLE> t(a, bid);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)t.j * kDropoutStep : 0;
  f32x4 s[CH], r[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) s[k] = t.get(a.x, k);
  if (a.residual) {
#pragma unroll
    for (int k = 0; k < CH; ++k) r[k] = t.get(a.residual, k);
  }
  double q[4] = {};
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (DROP) s[k] = t.drop(a.drop, z0, k, s[k]);
    if (a.residual) s[k] = r[k] + s[k];
    if (a.sum) t.put(a.sum, k, s[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double v = t.has(k) ? (double)s[k][e] : 0.0;
      q[e] = fma(v, v, q[e]);
    }
  }
  held_sums(q, t.row, part, sum);
  f32x4 rstd;
#pragma unroll
  for (int e = 0; e < 4; ++e) rstd[e] = inv_sqrt(q[e] * a.inv_f + a.eps);
  if (a.rstd && threadIdx.x < kHeldRows / 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < t.left) a.rstd[t.n0 + t.row + e] = rstd[e];
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) t.put(a.y, k, (s[k] * rstd) * t.of_column(a.gamma, k));
}
template <int CH, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_held_fwd_kernel(NormArgs a) {
  __shared__ double part[kNormWaves][kHeldRows], sum[kHeldRows];
  const int bid = held_tile(a);
  if ((int64_t)(bid + 1) * kHeldRows <= a.N) rms_norm_held_fwd_tile<CH, DROP, true>(a, bid, part, sum);
  else rms_norm_held_fwd_tile<CH, DROP, false>(a, bid, part, sum);
}

template <int CH, bool DROP, bool WHOLE>
__device__ __forceinline__ void rms_norm_held_bwd_tile(const NormArgs& a, int bid, double (*part)[kHeldRows], double* sum) {
  constexpr int P = CH < 4 ? CH : 4;  // of dsum under way
  const HeldSeat<WHOLE> t(a, bid);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)t.j * kDropoutStep : 0;
  f32x4 u[CH], d[CH], p[P], rstd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < t.left) rstd[e] = a.rstd[t.n0 + t.row + e];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    u[k] = t.get(a.s, k);
    d[k] = t.get(a.dy, k);
  }
  if (a.dsum) {
#pragma unroll
    for (int k = 0; k < P; ++k) p[k] = t.get(a.dsum, k);
  }
  __builtin_amdgcn_sched_barrier(0);
  double q[4] = {};
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const float g = t.has(k) ? t.of_column(a.gamma, k) : 0.f;
    float dg = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[k][e] *= rstd[e];
      if (e < t.left) dg = fmaf(d[k][e], u[k][e], dg);
      d[k][e] *= g;
      q[e] = t.has(k) ? fma((double)d[k][e], (double)u[k][e], q[e]) : q[e];
    }
    for (int o = kHeldRows / 8; o > 0; o >>= 1) dg += __shfl_xor(dg, o, 64);
    if (t.row == 0 && t.has(k)) (a.gamma_part + (int64_t)t.tile * a.F + t.column(k))[t.lane_f] = dg;
    __builtin_amdgcn_sched_barrier(0);
  }
  held_sums(q, t.row, part, sum);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    f32x4 g;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = rstd[e] * fmaf(-u[k][e], (float)(q[e] * a.inv_f), d[k][e]);
      if (a.dsum) g[e] += p[k % P][e];
    }
    if (a.dsum && k + P < CH) p[k % P] = t.get(a.dsum, k + P);
    __builtin_amdgcn_sched_barrier(0);
    if (a.dresidual) t.put(a.dresidual, k, g);
    t.put(a.dx, k, DROP ? t.drop(a.drop, z0, k, g) : g);
  }
}
template <int CH, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_held_bwd_kernel(NormArgs a) {
  __shared__ double part[kNormWaves][kHeldRows], sum[kHeldRows];
  const int bid = held_tile(a);
  if ((int64_t)(bid + 1) * kHeldRows <= a.N) rms_norm_held_bwd_tile<CH, DROP, true>(a, bid, part, sum);
  else rms_norm_held_bwd_tile<CH, DROP, false>(a, bid, part, sum);
}

// Features of a thread that a block of few rows holds: in the forward as many as need
// no second launch to be slower (8 x 2048: 9.7 us for 10.2 in tiles), in the backward, with
// two launches either way, what one block does as fast as many (32 x 128: 18.5 us with
// the forward for 20.9 in tiles, 32 x 512 26.7 and 21.0).
constexpr int kFewHeld = 16, kFewHeldBack = 4;
// Blocks of a large matrix: fewer leave CUs without work, more leave more sums for every
// block to join (4097 x 4099 both ways: 195 us with 256, 165 with 512 and 1024, 212 with
// 2193, a tile of 32 columns each).
constexpr int64_t kTileBlocks = 512;

// Few rows: up to 32, as many as a block holds of them.
bool few_rows(NormArgs& a, int held) {
  int shift = 0;
  while (((int64_t)1 << shift) < a.N && shift < 6) ++shift;
  if (a.N > 32 || (a.F << shift) > (int64_t)kNormThreads * held) return false;
  a.shift = shift;
  return true;
}

void set_tiles(NormArgs& a) {
  a.shift = 0;
  while (((int64_t)4 << a.shift) < a.N && a.shift < 6) ++a.shift;
  const int64_t rows = (int64_t)4 << a.shift, cols = (int64_t)K * (kTileThreads >> a.shift);
  const int64_t col_tiles = (a.F + cols - 1) / cols;
  a.row_tiles = (int)((a.N + rows - 1) / rows);
  const int64_t more = a.row_tiles * col_tiles / kTileBlocks;
  a.chunks = (int)(more < 2 ? 1 : more < col_tiles ? more : col_tiles);
  a.col_tiles = (int)((col_tiles + a.chunks - 1) / a.chunks);
}

// Rows held: at least the features that a wave has side by side, and at most as many as
// the registers of a block hold.  Forward in tiles and held, us, in a graph:
//   rows      512 features    768             1024
//   40        9.1 and 6.1     9.5 and 7.5     9.2 and 8.7
//   300       9.2 and 6.3     9.6 and 8.0     10.1 and 9.6
//   1000      9.7 and 6.7     10.4 and 8.5    11.1 and 10.5
//   2000      9.8 and 7.1     10.8 and 9.3    11.9 and 11.8
//   4000      11.1 and 8.2    15.8 and 11.0   19.9 and 13.9
//   8000      19.1 and 11.6   25.5 and 16.2   29.8 and 21.0
// Both ways in tiles and held: 8192 x 512 42.4 and 36.6, 1000 x 512 22.7 and 18.5, 8191 x 512
// 49 and 35, 131072 x 256 317 and 263, 8192 x 1024 94 and 67.  More than 512 features need
// as many registers as there are and one block's backward runs as long as two launches,
// so that few rows of them stay with tiles there (kernels' times: 1000 x 1024 13.5 and
// 15.8, 4096 x 1024 23.3 and 31.1, 6000 x 1024 35.4 and 28.5; of 513 to 1023 features it is
// not measured apart).  A backward in tiles behind a held forward takes some 2 us longer at
// 1000 x 1024 than behind one in tiles, 26.2 for 24.6 both ways, and no longer at 300 and
// 2000.
constexpr int kHeldFeatures = 1024;
bool rows_held(NormArgs& a, bool backward) {
  if (a.F < 256 / kHeldRows || a.F > kHeldFeatures || (backward && a.F > 512 && a.N < 6000)) return false;
  if (a.N >= (int64_t)1 << 26) return false;  // (a grid has fewer than 2^32 threads)
  a.row_tiles = (int)((a.N + kHeldRows - 1) / kHeldRows);
  return true;
}
// f(the times that a block's threads go through its features)
template <class F>
void with_passes(const NormArgs& a, F&& f) {
  const int n = (int)((a.F * kHeldRows + 4 * kNormThreads - 1) / (4 * kNormThreads));
  if (n <= 1) f(std::integral_constant<int, 1>{});
  else if (n <= 2) f(std::integral_constant<int, 2>{});
  else if (n <= 3) f(std::integral_constant<int, 3>{});
  else if (n <= 4) f(std::integral_constant<int, 4>{});
  else if (n <= 6) f(std::integral_constant<int, 6>{});
  else f(std::integral_constant<int, 8>{});
}

template <bool DROP>
int run_forward(NormArgs& a, hipStream_t st, const char* who) {
  const dim3 threads(kNormThreads);
  if (few_rows(a, kFewHeld)) {
    const int64_t per = ((a.F << a.shift) + kNormThreads - 1) / kNormThreads;
    if (per <= 4) hipLaunchKernelGGL((rms_norm_few_fwd_kernel<4, DROP>), dim3(1), threads, 0, st, a);
    else hipLaunchKernelGGL((rms_norm_few_fwd_kernel<kFewHeld, DROP>), dim3(1), threads, 0, st, a);
    return check_launch(who);
  }
  if (rows_held(a, false)) {
    with_passes(a, [&](auto n) {
      hipLaunchKernelGGL((rms_norm_held_fwd_kernel<n.value, DROP>), dim3((unsigned)a.row_tiles), threads, 0, st, a);
    });
    return check_launch(who);
  }
  set_tiles(a);
  const int64_t tiles = (int64_t)a.row_tiles * a.col_tiles;
  CNHIP_REQUIRE(tiles < ((int64_t)1 << 31), "%s: too large", who);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, (size_t)a.col_tiles * (size_t)a.N * sizeof(double), &ws, who));
  a.part = static_cast<double*>(ws);
  const dim3 grid((unsigned)tiles), tile_threads(kTileThreads);
  hipLaunchKernelGGL(rms_norm_sum_kernel<DROP>, grid, tile_threads, 0, st, a);
  CNHIP_TRY(check_launch(who));
  hipLaunchKernelGGL(rms_norm_apply_kernel<DROP>, grid, tile_threads, 0, st, a);
  return check_launch(who);
}

template <bool DROP>
int run_backward(NormArgs& a, hipStream_t st, const char* who) {
  const dim3 threads(kNormThreads);
  const bool few = few_rows(a, kFewHeldBack);
  a.row_tiles = a.col_tiles = a.chunks = 1;
  const bool held = !few && rows_held(a, true);
  if (!few && !held) set_tiles(a);
  const int64_t tiles = (int64_t)a.row_tiles * a.col_tiles, gamma_blocks = (a.F + 63) / 64;
  CNHIP_REQUIRE(tiles + gamma_blocks < ((int64_t)1 << 31), "%s: too large", who);
  const size_t sums = few || held ? 0 : (size_t)a.col_tiles * (size_t)a.N * sizeof(double);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, sums + (size_t)a.row_tiles * (size_t)a.F * sizeof(float), &ws, who));
  a.part = static_cast<double*>(ws);
  a.gamma_part = reinterpret_cast<float*>(static_cast<char*>(ws) + sums);
  if (few || held) {
    if (few) hipLaunchKernelGGL((rms_norm_few_bwd_kernel<kFewHeldBack, DROP>), dim3(1), threads, 0, st, a);
    else
      with_passes(a, [&](auto n) {
        hipLaunchKernelGGL((rms_norm_held_bwd_kernel<n.value, DROP>), dim3((unsigned)a.row_tiles), threads, 0, st, a);
      });
    CNHIP_TRY(check_launch(who));
    hipLaunchKernelGGL(rms_norm_gamma_kernel, dim3((unsigned)((a.F + 15) / 16)), threads, 0, st, a);
    return check_launch(who);
  }
  const dim3 grid((unsigned)tiles), more((unsigned)(tiles + gamma_blocks)), tile_threads(kTileThreads);
  hipLaunchKernelGGL(rms_norm_dots_kernel, grid, tile_threads, 0, st, a);
  CNHIP_TRY(check_launch(who));
  hipLaunchKernelGGL(rms_norm_grad_kernel<DROP>, more, tile_threads, 0, st, a);
  return check_launch(who);
}

int check_drop(float p, const char* who) {
  CNHIP_REQUIRE(p >= 0.0f && p < 1.0f, "%s: drop probability %g outside [0, 1)", who, (double)p);
  return CNHIP_OK;
}
Drop drop_of(float p, uint64_t seed, uint64_t offset, const uint64_t* counter) {
  return Drop{dropout_limit(p), 1.0f / (1.0f - p), seed, offset, counter};
}
int check_shape(int64_t N, int64_t F, const char* who) {
  CNHIP_REQUIRE(N > 0 && F > 0, "%s: bad shape N=%lld F=%lld", who, (long long)N, (long long)F);
  CNHIP_REQUIRE(N < ((int64_t)1 << 28) && F < ((int64_t)1 << 24), "%s: too large", who);
  return CNHIP_OK;
}

}  // namespace
}  // namespace cnhip

extern "C" {

int cnhip_dropout_seeded(const float* x, float* y, int64_t n, float p, uint64_t seed, uint64_t offset,
                         const uint64_t* counter, cnhip_stream_t stream) {
  const char* who = "cnhip_dropout_seeded";
  CNHIP_REQUIRE(n >= 0, "%s: negative size", who);
  CNHIP_TRY(cnhip::check_drop(p, who));
  if (n == 0) return CNHIP_OK;
  CNHIP_REQUIRE(x && y, "%s: NULL pointer", who);
  const hipStream_t st = cnhip::as_stream(stream);
  cnhip::HbmTimer timer("dropout_seeded_kernel", 8.0 * (double)n, st);
  hipLaunchKernelGGL(cnhip::dropout_seeded_kernel, dim3(cnhip::elementwise_grid((n + 3) / 4, 256)), dim3(256), 0, st, x,
                     y, n, cnhip::drop_of(p, seed, offset, counter));
  return cnhip::check_launch(who);
}

int cnhip_dropout_advance(uint64_t* counter, uint64_t n, cnhip_stream_t stream) {
  const char* who = "cnhip_dropout_advance";
  CNHIP_REQUIRE(counter, "%s: NULL pointer", who);
  hipLaunchKernelGGL(cnhip::dropout_advance_kernel, dim3(1), dim3(1), 0, cnhip::as_stream(stream), counter, n);
  return cnhip::check_launch(who);
}

int cnhip_rms_norm_forward(const float* x, const float* residual, const float* gamma, float* y, float* sum,
                           float* rstd, int64_t N, int64_t F, float eps, float p, uint64_t seed, uint64_t offset,
                           const uint64_t* counter, cnhip_stream_t stream) {
  const char* who = "cnhip_rms_norm_forward";
  CNHIP_TRY(cnhip::check_shape(N, F, who));
  CNHIP_TRY(cnhip::check_drop(p, who));
  CNHIP_REQUIRE(eps > 0.f && std::isfinite(eps), "%s: eps must be positive and finite, got %g", who, (double)eps);
  CNHIP_REQUIRE(x && gamma && y, "%s: NULL pointer", who);
  cnhip::NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.gamma = gamma;
  a.y = y;
  a.sum = sum;
  a.rstd = rstd;
  a.N = N;
  a.F = F;
  a.eps = (double)eps;
  a.inv_f = 1.0 / (double)F;
  a.drop = cnhip::drop_of(p, seed, offset, counter);
  const hipStream_t st = cnhip::as_stream(stream);
  cnhip::HbmTimer timer("rms_norm_fwd_kernel", 4.0 * (double)N * (double)F * (2 + (residual != nullptr) + (sum != nullptr)),
                        st);
  return p > 0.f ? cnhip::run_forward<true>(a, st, who) : cnhip::run_forward<false>(a, st, who);
}

int cnhip_rms_norm_backward(const float* sum, const float* rstd, const float* gamma, const float* dy, const float* dsum,
                            float* dx, float* dresidual, float* dgamma, int64_t N, int64_t F, float p, uint64_t seed,
                            uint64_t offset, const uint64_t* counter, int accumulate, cnhip_stream_t stream) {
  const char* who = "cnhip_rms_norm_backward";
  CNHIP_TRY(cnhip::check_shape(N, F, who));
  CNHIP_TRY(cnhip::check_drop(p, who));
  CNHIP_REQUIRE(sum && rstd && gamma && dy && dx && dgamma, "%s: NULL pointer", who);
  CNHIP_REQUIRE(accumulate == 0 || accumulate == 1, "%s: accumulate must be 0 or 1", who);
  cnhip::NormArgs a{};
  a.s = sum;
  a.rstd = const_cast<float*>(rstd);
  a.gamma = gamma;
  a.dy = dy;
  a.dsum = dsum;
  a.dx = dx;
  a.dresidual = dresidual;
  a.dgamma = dgamma;
  a.N = N;
  a.F = F;
  a.inv_f = 1.0 / (double)F;
  a.drop = cnhip::drop_of(p, seed, offset, counter);
  a.accumulate = accumulate;
  const hipStream_t st = cnhip::as_stream(stream);
  cnhip::HbmTimer timer("rms_norm_bwd_kernel",
                        4.0 * (double)N * (double)F * (3 + (dsum != nullptr) + (dresidual != nullptr)), st);
  return p > 0.f ? cnhip::run_backward<true>(a, st, who) : cnhip::run_backward<false>(a, st, who);
}

}  // extern "C"
