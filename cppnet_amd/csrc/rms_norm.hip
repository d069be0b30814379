// Root-mean-square norm of a residual's sum, and dropout whose mask is never
// stored.
//
//   s = residual + drop(x),  rstd_n = 1 / sqrt(mean_f s_nf^2 + eps),
//   y_nf = s_nf rstd_n gamma_f
// backward, n_nf = s_nf rstd_n, d_nf = gamma_f dy_nf:
//   ds = dsum + rstd (d - n mean_f(d n)),  dresidual = ds, dx = drop(ds),
//   dgamma_f (+)= sum_n dy_nf n_nf
//
// Matrices are ColMajor [N, F]: the features of a row lie N apart, so a block
// takes a few rows side by side and all of their features, and holds them in
// registers between the sum over the features and the result.  Everything is
// read once and written once.  The sums over a row are kept in 64 bits, which
// neither overflow nor vanish for any finite fp32 row.
//
// Element j of the [N, F] storage is kept where the generator's word for
// position + j says so; the backward draws the same words again.
#include <hip/hip_runtime.h>

#include <cmath>

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
  float *dx, *dresidual, *dgamma, *part;
  int64_t N, F;
  int shift;       // log2 of the rows of a block
  int64_t tiles;   // of that many rows
  double eps, inv_f;
  Drop drop;
  int accumulate;
};

constexpr int kNormThreads = 1024, kNormWaves = kNormThreads / 64;

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

// 1 / sqrt(v) to fp32's precision and range.
__device__ __forceinline__ float inv_sqrt(double v) {
  double r = __builtin_amdgcn_rsq(v);
  r = r * fma(-0.5 * v * r, r, 1.5);
  return (float)r;
}

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

// K: a thread's features at a time.  ONCE: they are all of its features; otherwise s is
// read again for the result.
template <int K, bool ONCE, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_fwd_kernel(NormArgs a) {
#pragma clang fp contract(off)
  __shared__ double part[kNormWaves][64];
  const Seat w(a.N, a.shift);
  const int64_t n0 = (int64_t)blockIdx.x << a.shift;
  const bool in = n0 + w.r < a.N;
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)w.j * kDropoutStep : 0;
  const int rounds = (int)((a.F + w.cols - 1) / w.cols);  // of all the columns of threads
  auto get = [&](int k) {
    const int64_t o = n0 + w.part(k);
    float v = (a.x + o)[w.j];
    if (DROP) v = dropped(a.drop, z0 + (uint64_t)o * kDropoutStep, v);
    return a.residual ? (a.residual + o)[w.j] + v : v;
  };
  float s[K];
  double q = 0.0;
  for (int k0 = 0; k0 < rounds; k0 += K) {
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = in && w.has(k0 + k, a.F) ? get(k0 + k) : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      q = fma((double)s[k], (double)s[k], q);
      if (a.sum && in && w.has(k0 + k, a.F)) (a.sum + n0 + w.part(k0 + k))[w.j] = s[k];
    }
    if (ONCE) break;
  }
  const float rstd = inv_sqrt(row_sum(q, a.shift, part) * a.inv_f + a.eps);
  if (!in) return;
  if (a.rstd && threadIdx.x < (unsigned)w.rows) a.rstd[n0 + w.r] = rstd;
  for (int k0 = 0; k0 < rounds; k0 += K) {
    if (!ONCE) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        s[k] = w.has(k0 + k, a.F) ? (a.sum ? (a.sum + n0 + w.part(k0 + k))[w.j] : get(k0 + k)) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (w.has(k0 + k, a.F))
        (a.y + n0 + w.part(k0 + k))[w.j] = (s[k] * rstd) * (a.gamma + w.first0 + (int64_t)(k0 + k) * w.cols)[w.lane_f];
    if (ONCE) break;
  }
}

// A block takes every gridDim.x-th tile of rows and sums its part of dgamma over
// them: in registers where a thread's features are all at hand (ONCE).
template <int K, bool ONCE, bool DROP>
__global__ void __launch_bounds__(kNormThreads) rms_norm_bwd_kernel(NormArgs a) {
  __shared__ double part[2][kNormWaves][64];
  const Seat w(a.N, a.shift);
  const uint64_t z0 = DROP ? first_word(a.drop) + (uint64_t)w.j * kDropoutStep : 0;
  const int rounds = (int)((a.F + w.cols - 1) / w.cols);
  float dg[K];
#pragma unroll
  for (int k = 0; k < K; ++k) dg[k] = 0.f;
  int parity = 0;
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, parity ^= 1) {
    const int64_t n0 = tile << a.shift;
    const bool in = n0 + w.r < a.N;
    const float rstd = in ? a.rstd[n0 + w.r] : 0.f;
    float u[K], d[K];  // the normed row, and the gradient at it
    double q = 0.0;
    auto gamma = [&](int k) { return (a.gamma + w.first0 + (int64_t)k * w.cols)[w.lane_f]; };
    auto get = [&](int k0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const bool on = in && w.has(k0 + k, a.F);
        const int64_t o = n0 + w.part(k0 + k);
        u[k] = on ? (a.s + o)[w.j] * rstd : 0.f;
        d[k] = on ? (a.dy + o)[w.j] : 0.f;
      }
    };
    for (int k0 = 0; k0 < rounds; k0 += K) {
      get(k0);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (ONCE) dg[k] = fmaf(d[k], u[k], dg[k]);
        d[k] *= w.has(k0 + k, a.F) ? gamma(k0 + k) : 0.f;
        q = fma((double)d[k], (double)u[k], q);
      }
      if (ONCE) break;
    }
    const float c = (float)(row_sum(q, a.shift, part[parity]) * a.inv_f);
    for (int k0 = 0; k0 < rounds; k0 += K) {
      if (!ONCE) {
        get(k0);
#pragma unroll
        for (int k = 0; k < K; ++k) d[k] *= w.has(k0 + k, a.F) ? gamma(k0 + k) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!in || !w.has(k0 + k, a.F)) continue;
        const int64_t o = n0 + w.part(k0 + k);
        float g = rstd * fmaf(-u[k], c, d[k]);
        if (a.dsum) g += (a.dsum + o)[w.j];
        if (a.dresidual) (a.dresidual + o)[w.j] = g;
        (a.dx + o)[w.j] = DROP ? dropped(a.drop, z0 + (uint64_t)o * kDropoutStep, g) : g;
      }
      if (ONCE) break;
    }
  }
  if (!ONCE) return;
  // over the rows of the block: lanes side by side
#pragma unroll
  for (int k = 0; k < K; ++k) {
    for (int o = w.rows >> 1; o > 0; o >>= 1) dg[k] += __shfl_xor(dg[k], o, 64);
    if (w.r == 0 && w.has(k, a.F)) (a.part + (int64_t)blockIdx.x * a.F + w.first0 + (int64_t)k * w.cols)[w.lane_f] = dg[k];
  }
}

// dgamma (+)= the blocks' parts, in order: 64 features a block, its waves share the parts.
__global__ void __launch_bounds__(1024) rms_norm_gamma_kernel(const float* __restrict__ part, float* dgamma, int64_t F,
                                                              int blocks, int accumulate) {
  __shared__ float sum[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f = (int64_t)blockIdx.x * 64 + lane;
  float t = 0.f;
  if (f < F) {
#pragma unroll 8
    for (int b = wave; b < blocks; b += 16) t += part[(int64_t)b * F + f];
  }
  sum[wave][lane] = t;
  __syncthreads();
  if (wave || f >= F) return;
  for (int w = 1; w < 16; ++w) t += sum[w][lane];
  dgamma[f] = accumulate ? dgamma[f] + t : t;
}

// dgamma of wide rows, from dy, s and rstd once more: a wave for a feature's rows.
__global__ void __launch_bounds__(256) rms_norm_gamma_wide_kernel(NormArgs a) {
  __shared__ float sum[4];
  const int64_t f = blockIdx.x;
  const float *s = a.s + a.N * f, *dy = a.dy + a.N * f;
  float t = 0.f;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < a.N; n += 256) t = fmaf(dy[n], s[n] * a.rstd[n], t);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x) return;
  t = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  a.dgamma[f] = a.accumulate ? a.dgamma[f] + t : t;
}

constexpr int kNormHeld = 32, kNormHeldBack = 16;  // features of a thread that are kept between the passes
constexpr int kNormBlocks = 512;    // of the backward, and so parts of dgamma at most

// Rows of a block, as a power of two: 32 are whole lines of memory.  Fewer where there
// are fewer rows, or where 32 rows are more than a block holds.
int rows_shift(int64_t N, int64_t F, int held) {
  int shift = 5;
  while (shift > 0 && ((int64_t)1 << (shift - 1)) >= N) --shift;
  while (shift > 4 && (F << shift) > (int64_t)kNormThreads * held) --shift;
  return shift;
}

template <bool BWD, bool DROP>
int run_norm(NormArgs& a, hipStream_t st, const char* who) {
  constexpr int held = BWD ? kNormHeldBack : kNormHeld;
  a.shift = rows_shift(a.N, a.F, held);
  a.tiles = (a.N + ((int64_t)1 << a.shift) - 1) >> a.shift;
  const int64_t cols = kNormThreads >> a.shift, per = (a.F + cols - 1) / cols;
  const bool once = per <= held;
  if constexpr (!BWD) {
    const dim3 grid((unsigned)a.tiles), threads(kNormThreads);
    if (per <= 4) hipLaunchKernelGGL((rms_norm_fwd_kernel<4, true, DROP>), grid, threads, 0, st, a);
    else if (per <= 16) hipLaunchKernelGGL((rms_norm_fwd_kernel<16, true, DROP>), grid, threads, 0, st, a);
    else if (once) hipLaunchKernelGGL((rms_norm_fwd_kernel<kNormHeld, true, DROP>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((rms_norm_fwd_kernel<16, false, DROP>), grid, threads, 0, st, a);
    return check_launch(who);
  } else {
    const int blocks = (int)(a.tiles < kNormBlocks ? a.tiles : kNormBlocks);
    const dim3 grid((unsigned)blocks), threads(kNormThreads);
    if (once) {
      void* ws = nullptr;
      CNHIP_TRY(scratch(st, kScratchLayer, (size_t)blocks * (size_t)a.F * sizeof(float), &ws, who));
      a.part = static_cast<float*>(ws);
    }
    if (per <= 4) hipLaunchKernelGGL((rms_norm_bwd_kernel<4, true, DROP>), grid, threads, 0, st, a);
    else if (once) hipLaunchKernelGGL((rms_norm_bwd_kernel<kNormHeldBack, true, DROP>), grid, threads, 0, st, a);
    else hipLaunchKernelGGL((rms_norm_bwd_kernel<16, false, DROP>), grid, threads, 0, st, a);
    CNHIP_TRY(check_launch(who));
    if (once)
      hipLaunchKernelGGL(rms_norm_gamma_kernel, dim3((unsigned)((a.F + 63) / 64)), dim3(1024), 0, st, a.part, a.dgamma,
                         a.F, blocks, a.accumulate);
    else
      hipLaunchKernelGGL(rms_norm_gamma_wide_kernel, dim3((unsigned)a.F), dim3(256), 0, st, a);
    return check_launch(who);
  }
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
  CNHIP_REQUIRE(N < ((int64_t)1 << 28) && F < ((int64_t)1 << 31), "%s: too large", who);
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
  return p > 0.f ? cnhip::run_norm<false, true>(a, st, who) : cnhip::run_norm<false, false>(a, st, who);
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
  return p > 0.f ? cnhip::run_norm<true, true>(a, st, who) : cnhip::run_norm<true, false>(a, st, who);
}

}  // extern "C"
