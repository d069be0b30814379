// A gated feed-forward layer: two projections, an activation of the first and
// the product with the second, in one call, and its backward pass.
//
//   Z = X W + b, gate = Z[:, :F], up = Z[:, F:],  H = act(gate) up
// backward:
//   dgate = dH up act'(gate), dup = dH act(gate), dZ = [dgate dup],
//   dX = dZ W^T,  dW (+)= X^T dZ,  db (+)= column sums of dZ
//
// Products of many rows run on the fp16 matrix cores over operands packed as pairs
// (mfma_pair.hpp).  W's columns are packed in blocks of 32, a gate's and then its
// up's, so one wave's accumulators hold both values of an element and the
// activation and the product are done where the sums are.  dZ is packed in the
// same order of columns straight from Z and dH, and serves both products of the
// backward, once along its columns and once along its rows.
//
// Bound by the fp16 matrix cores at the clock that the power limit leaves, which differs
// from card to card.  8192 rows, 1024 -> 4096, GELU: forward 411 to 490 us (280 to 334
// TFLOP/s of fp32 products, where a third of a library's fp16 rate is 387) and packing 38;
// back 711 to 813 (338 to 387), packing 152 (5.3 TB/s) and the bound of dZ 100 (4.7 TB/s).
// Few tiles by latency and what is moved between the launches: 1021 rows, 513 -> 1365, 9 +
// 21.5 us forward and 9.3 + 10.8 + 36 + 4.5 back.  Few rows by W: 4 rows, 512 -> 2048 4.7 us.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "act_math.hpp"
#include "common.hpp"
#include "mfma_pair.hpp"

namespace cnhip {
namespace {

using pr::f32x16;
using pr::f32x4;
using pr::f32x4u;

// Largest finite values, as bits: of W, of a piece's X and half a bound of its dZ.
struct FfnScales {
  uint32_t w, x, z;
};
// The products' tiles.  The forward's are Half, two to a CU, of which one stores while the
// other computes, which leaves less of a call's grid empty (half and whole tiles, us: 1021 x
// 513 -> 1365 both directions 103.6 and 108.7, 256 x 1024 -> 4096 50 and 55, 8192 x 1024 ->
// 4096 393 and 386), or Small; the backward's Whole (half tiles across the rows of both
// operands need more registers than there are) or Small: where there are few tiles these
// need fewer splits or none and pad less, and a step of them costs half as much again for
// a product (Small and the others, kernels with the joining of splits, us: 1021 x 513 ->
// 1365 forward 21 and 30, back 40 and 50; 1024 x 512 -> 2048 22 and 32.5, 41 and 60; 512 x
// 512 -> 2048 back 27 and 38; 2048 x 1024 -> 4096 127 and 104, 227 and 207).
using Half = pr::Tile<2>;
using Whole = pr::Tile<4>;
using Small = pr::Tile<2, 2, 2>;
// What the blocks that look for them found: of W, X and dZ.
constexpr int kMaxBlocks[3] = {256, 256, 512};
constexpr int kMaxAt[3] = {0, 256, 512}, kMaxParts = 1024;

struct FfnArgs {
  const float *X, *W, *b, *Z, *dH;
  float *H, *Zout;
  int64_t N, D, F;
  int64_t row0, R;     // the piece's rows (backward)
  int act;
  char *xp, *wp, *zp;  // packed X [rows x D], W^T [2 Fp x D], dZ [rows x 2 Fp]
  int *xe, *we;        // forward: the exponents of a row of X, of 32 rows of W^T
  int steps_d;         // of 16 features of D
  int steps_f;         // of 16 of the hidden features
  uint32_t* max_part;  // [kMaxParts]
  int max_blocks[3];
  FfnScales* scales;
  int z_blocks;        // blocks of 32 rows that a wave packs of dZ
  float* db_part;      // [ceil(R / 32 / z_blocks)][2 F], or null
};

// Column of W that row m of the packed W^T holds; -1 for padding.
__device__ __forceinline__ int64_t column_of(int64_t m, int64_t F) {
  const int64_t j = (m >> 6) * 32 + (m & 31);
  return j < F ? (m & 32 ? F : 0) + j : -1;
}

__device__ __forceinline__ void sigmoid_parts(float z, float& on, float& off) {
  const float e = exp_acc(-fminf(fabsf(z), 200.f)), r = __builtin_amdgcn_rcpf(1.f + e);
  on = z >= 0.f ? r : e * r;
  off = z >= 0.f ? e * r : r;
  if (z != z) on = off = z;
}
// Phi(z), and exp(-z^2 / 2); beyond 200 it is 0 or 1, and the square would leave fp32's range.
__device__ __forceinline__ float gate_cdf(float z, float& e) {
  return ncdf_f(z, fminf(fabsf(z), 200.f) * 0.70710678118654752440f, &e);
}
// act(z)
__device__ __forceinline__ float gate_f(int act, float z) {
  if (act == CNHIP_GATE_GELU) {
    float e;
    return z * gate_cdf(z, e);
  }
  if (act == CNHIP_GATE_RELU) return relu_f(z);
  float on, off;
  sigmoid_parts(z, on, off);
  return act == CNHIP_GATE_SILU ? z * on : on;
}
// act(z) and act'(z)
__device__ __forceinline__ void gate_both(int act, float z, float& y, float& d) {
  if (act == CNHIP_GATE_GELU) {
    float e;
    const float cdf = gate_cdf(z, e);
    y = z * cdf;
    d = fmaf(z, 0.39894228040143267794f * e, cdf);
    return;
  }
  if (act == CNHIP_GATE_RELU) {
    y = relu_f(z);
    d = relu_mask(y);
    return;
  }
  float on, off;
  sigmoid_parts(z, on, off);
  y = act == CNHIP_GATE_SILU ? z * on : on;
  d = act == CNHIP_GATE_SILU ? on * fmaf(z, off, 1.f) : on * off;
}

// f(act), act a constant
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == CNHIP_GATE_SILU) f(std::integral_constant<int, CNHIP_GATE_SILU>{});
  else if (act == CNHIP_GATE_GELU) f(std::integral_constant<int, CNHIP_GATE_GELU>{});
  else if (act == CNHIP_GATE_SIGMOID) f(std::integral_constant<int, CNHIP_GATE_SIGMOID>{});
  else f(std::integral_constant<int, CNHIP_GATE_RELU>{});
}

// ------------------------------------------------------------------ forward
// X and W^T packed, every row of X and every 32 rows of W^T with an exponent of
// their own: a block of sixteen waves for 32 rows, which keep their first kHeld steps
// and read the others twice (the second time from the L2).
__global__ void __launch_bounds__(1024) ffn_pack_own_kernel(FfnArgs a, int w_blocks) {
  constexpr int kHeld = 4;
  __shared__ uint32_t part[16][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const bool w = (int)blockIdx.x < w_blocks;
  const int64_t blk = w ? blockIdx.x : (int64_t)blockIdx.x - w_blocks, row = blk * 32 + r;
  const int64_t col = w ? column_of(row, a.F) : 0;
  const bool in = w ? col >= 0 : row < a.N;
  auto load = [&](int step, float (&x)[8]) {
    const int64_t d0 = step * 16 + 8 * h;
    if (step >= a.steps_d) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    } else if (w) {
      const float* p = a.W + col * a.D + d0;
      if (in && d0 + 8 <= a.D) {
        const f32x4 lo = *reinterpret_cast<const f32x4u*>(p), hi = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = lo[e];
          x[4 + e] = hi[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = in && d0 + e < a.D ? p[e] : 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = in && d0 + e < a.D ? a.X[row + a.N * (d0 + e)] : 0.f;
    }
  };
  uint32_t m = 0;
  float held[kHeld][8];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) load(wave + 16 * u, held[u]);
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, pr::finite_bits(held[u][e]));
  for (int s0 = wave + 16 * kHeld; s0 < a.steps_d; s0 += 32) {
    float x[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) load(s0 + 16 * u, x[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, pr::finite_bits(x[u][e]));
  }
  if (w) m = pr::wave_max(m);
  else m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  if (lane < 32) part[wave][lane] = m;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 16; ++q) m = max(m, part[q][r]);
  const int exp = pr::scale_exp(m);
  const float f = pr::exp2i(exp);
  if (wave == 0 && lane < 32) {
    if (!w && in) a.xe[row] = exp;
    if (w && lane == 0) a.we[blk] = exp;
  }
  auto put = [&](int step, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f;
    pr::put_frag(w ? a.wp : a.xp, blk, a.steps_d, step, x);
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (wave + 16 * u < a.steps_d) put(wave + 16 * u, held[u]);
  for (int step = wave + 16 * kHeld; step < a.steps_d; step += 16) {
    float x[8];
    load(step, x);
    put(step, x);
  }
}

// A: W^T (M: packed columns), B: X (N: rows); H and, where it is kept, Z.
template <class T>
__global__ void __launch_bounds__(T::NT, 2) ffn_forward_kernel(pr::GemmArgs g, FfnArgs a, float* part) {
  __shared__ __align__(16) char lds[T::kLds];
  int tm, tn;
  pr::tile_of((int)blockIdx.x, (g.M + T::TM - 1) / T::TM, (g.N + T::TN - 1) / T::TN, tm, tn);
  pr::AccOf<T::MI> acc;
  const int t0 = (int)blockIdx.y * g.steps_per_split;
  pr::gemm_tile<false, false, T>(g, tm, tn, t0, min(g.steps, t0 + g.steps_per_split), lds, acc);
  if (part) {
    pr::put_tile<false, T>(acc, tm, tn, g.M, g.N, part + (int64_t)blockIdx.y * g.M * g.N, g.N, [](float x) { return x; });
    return;
  }
  const int lane = threadIdx.x & 63;
  const int block0 = (tm * T::TM + T::row0()) / 32;  // the wave's first of 32 packed columns: a gate's
  const int64_t n0 = (int64_t)tn * T::TN + T::column(0);
  // A test for every element would end the run of loads, functions and stores behind it
  // (in tiles of 256 x 128: 1024 rows, 64 -> 1024 24 us for 12; 8192 rows, 1024 -> 4096 475 us
  // for 411), so the activation and whole tiles are told apart here.
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < T::MI; i += 2) {
      if (block0 + i >= g.M / 32) break;
      const int64_t first = (int64_t)(block0 + i) * 16, f0 = first + 4 * (lane >> 5);
      const bool whole = first + 32 <= a.F && n0 - (lane & 31) + 32 * T::J <= a.N;
      auto row = [](int e) { return 8 * (e / 4) + e % 4; };
      float bg[16], bu[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t f = f0 + row(e) < a.F ? f0 + row(e) : a.F - 1;
        bg[e] = a.b ? a.b[f] : 0.f;
        bu[e] = a.b ? a.b[a.F + f] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < T::J; ++j) {
        const int64_t n = n0 + 32 * j;
        const int ex = a.xe[n < a.N ? n : a.N - 1], eg = -ex - a.we[block0 + i], eu = -ex - a.we[block0 + i + 1];
        float h[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          acc.x[i][j][e] = pr::times_exp2(acc.x[i][j][e], eg) + bg[e];
          acc.x[i + 1][j][e] = pr::times_exp2(acc.x[i + 1][j][e], eu) + bu[e];
          h[e] = gate_f(act, acc.x[i][j][e]) * acc.x[i + 1][j][e];
        }
        float* to = a.H + n + a.N * f0;
        float* zg = a.Zout + n + a.N * f0;
        float* zu = zg + a.N * a.F;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 16; ++e) to[a.N * row(e)] = h[e];
          if (!a.Zout) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e) zg[a.N * row(e)] = acc.x[i][j][e];
#pragma unroll
          for (int e = 0; e < 16; ++e) zu[a.N * row(e)] = acc.x[i + 1][j][e];
        } else if (n < a.N) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (f0 + row(e) >= a.F) continue;
            to[a.N * row(e)] = h[e];
            if (!a.Zout) continue;
            zg[a.N * row(e)] = acc.x[i][j][e];
            zu[a.N * row(e)] = acc.x[i + 1][j][e];
          }
        }
      }
    }
  });
}

// The same from split sums, [splits][M][N].
__global__ void __launch_bounds__(256) ffn_join_kernel(FfnArgs a, const float* __restrict__ part, int64_t M, int splits) {
  const int64_t total = M * a.N;
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, f = blockIdx.y;
  if (n >= a.N) return;
  const int64_t at = ((f >> 5) * 64 + (f & 31)) * a.N + n;
  float gate = 0.f, up = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    gate += part[s * total + at];
    up += part[s * total + at + 32 * a.N];
  }
  const int ex = a.xe[n], blk = (int)(f >> 5) * 2;
  gate = pr::times_exp2(gate, -ex - a.we[blk]) + (a.b ? a.b[f] : 0.f);
  up = pr::times_exp2(up, -ex - a.we[blk + 1]) + (a.b ? a.b[a.F + f] : 0.f);
  if (a.Zout) {
    a.Zout[n + a.N * f] = gate;
    a.Zout[n + a.N * (a.F + f)] = up;
  }
  a.H[n + a.N * f] = gate_f(a.act, gate) * up;
}

// Few rows: each value of W is used for a handful of products, so the fp32 matrix
// cores keep up with memory and nothing is packed.  A block takes 8 hidden features
// (16 columns of W, the rows of the 16 x 16 tiles) and up to 128 rows; its eight waves
// share out D and meet in LDS.
// Packed, a call takes about 12 us more for its launches and 3.6 us for every million of D
// F to pack W, but a quarter of the time for a row's products.  This way and packed, us:
// 128 rows, 512 -> 2048 11.1 and 25, 1024 -> 4096 40 and 44; 256 rows, 512 -> 2048 22 and
// 26.7; 384 rows 35 and 27.5; 512 rows, 512 -> 1024 21.8 and 24; 1024 rows, 256 -> 512 12.4
// and 16.8, 2048 rows 21.4 and 18.1.
constexpr int kFewBlock = 128;
bool few_rows(int64_t N, int64_t D, int64_t F) {
  const double rows = (double)(N <= 64 ? (N + 15) / 16 * 16 : (N + kFewBlock - 1) / kFewBlock * kFewBlock);
  return N <= 65535 * (int64_t)kFewBlock && 1e-6 * (double)D * (double)F * (0.05 * rows - 3.6) <= 12.0;
}
template <int NB>
__global__ void __launch_bounds__(512) ffn_few_kernel(FfnArgs a) {
  __shared__ float part[8][16][16 * NB + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 8, f = f0 + (r & 7);
  const float* w = a.W + ((r >> 3) * a.F + (f < a.F ? f : a.F - 1)) * a.D;
  const int64_t n0 = (int64_t)blockIdx.y * kFewBlock;
  const float* X = a.X + n0;
  const int N = (int)(a.N - n0 < 16 * NB ? a.N - n0 : 16 * NB);
  f32x4 acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = NB > 4 ? 1 : NB > 2 ? 2 : 4;  // steps of 16 features under way
  for (int64_t d0 = 16 * wave; d0 < a.D; d0 += 128 * U) {
    f32x4 wv[U];
    float xv[U][NB][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t d = d0 + 128 * u + 4 * q;
      if (d + 4 <= a.D) {
        wv[u] = *reinterpret_cast<const f32x4u*>(w + d);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) wv[u][e] = d + e < a.D ? w[d + e] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          xv[u][j][e] = d + e < a.D && 16 * j + r < N ? X[16 * j + r + a.N * (d + e)] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < NB; ++j)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[u][e], xv[u][j][e], acc[j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][4 * q + e][16 * j + r] = acc[j][e];
  __syncthreads();
  for (int t = threadIdx.x; t < 8 * 16 * NB; t += 512) {
    const int n = t % (16 * NB), k = t / (16 * NB);
    if (n >= N || f0 + k >= a.F) continue;
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      gate += part[s][k][n];
      up += part[s][8 + k][n];
    }
    if (a.b) {
      gate += a.b[f0 + k];
      up += a.b[a.F + f0 + k];
    }
    const int64_t at = n0 + n + a.N * (f0 + k);
    if (a.Zout) {
      a.Zout[at] = gate;
      a.Zout[at + a.N * a.F] = up;
    }
    a.H[at] = gate_f(a.act, gate) * up;
  }
}

// ----------------------------------------------------------------- backward
__device__ __forceinline__ void grads_of(const FfnArgs& a, float gate, float up, float dh, float& dg, float& du) {
  float y, d;
  gate_both(a.act, gate, y, d);
  dg = dh * up * d;
  du = dh * y;
}

// dZ, [N, 2 F] as Z is stored: 4 values a thread.
__global__ void __launch_bounds__(256) ffn_dz_kernel(FfnArgs a, float* __restrict__ dZ) {
  const int64_t n = a.N * a.F, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int left = n - i < 4 ? (int)(n - i) : 4;
  f32x4 zg = {0.f, 0.f, 0.f, 0.f}, zu = zg, dh = zg;
  if (left == 4) {
    zg = *reinterpret_cast<const f32x4u*>(a.Z + i);
    zu = *reinterpret_cast<const f32x4u*>(a.Z + n + i);
    dh = *reinterpret_cast<const f32x4u*>(a.dH + i);
  } else {
    for (int e = 0; e < left; ++e) {
      zg[e] = a.Z[i + e];
      zu[e] = a.Z[n + i + e];
      dh[e] = a.dH[i + e];
    }
  }
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y, d;
      gate_both(act, zg[e], y, d);
      zg[e] = dh[e] * zu[e] * d;
      zu[e] = dh[e] * y;
    }
  });
  if (left == 4) {
    *reinterpret_cast<f32x4u*>(dZ + i) = zg;
    *reinterpret_cast<f32x4u*>(dZ + n + i) = zu;
  } else {
    for (int e = 0; e < left; ++e) {
      dZ[i + e] = zg[e];
      dZ[n + i + e] = zu[e];
    }
  }
}

// An upper bound of |dgate| and |dup|, up to twice dup's size and six times dgate's but next
// to a zero of act': an operand's scale need not be closer, and with the functions
// themselves the pass over Z and dH takes longer (8192 x 4096, GELU: 106 us for 99; 1021 x
// 1365, SiLU: 10.6 for 9.3).
//   z >= 0: |act| <= z (sigmoid: 1), |act'| <= 1.13
//   z < 0:  with r = e^z, or e^(-z^2 / 2) for GELU, |act| <= r |z|, |act'| <= r (1 + |z|);
//   GELU: Phi(z) <= r / 2 and |z| Phi(z) <= r / sqrt(2 pi), so |act| <= r min(|z| / 2, 0.4)
//   (r |z| is 2.5 |z| times it far out);
//   sigmoid: act <= r, and act' <= e^-|z| everywhere.  ReLU: as they are.
// Half of it is kept: the whole may lie past fp32's range where the gradient does not, and
// a bound that is not finite does not count.
__device__ __forceinline__ uint32_t half_grad_bound(int act, float gate, float up, float dh) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float m = fabsf(gate);
  float y, d;
  if (act == CNHIP_GATE_RELU) {
    y = 0.5f * relu_f(gate);
    d = 0.5f * relu_mask(gate);
  } else {
    const float r = 0.5f * __builtin_amdgcn_exp2f(-kLog2e * (act == CNHIP_GATE_GELU ? 0.5f * m * m : m));
    if (act == CNHIP_GATE_SIGMOID) {
      y = gate < 0.f ? r : 0.5f;
      d = r;
    } else {
      y = gate < 0.f ? r * (act == CNHIP_GATE_GELU ? fminf(0.5f * m, 0.4f) : m) : 0.5f * gate;
      d = gate < 0.f ? fmaf(r, m, r) : 0.5f * 1.13f;
    }
  }
  return max(pr::finite_bits(dh * up * d), pr::finite_bits(dh * y));
}
// dZ's exponent from the largest of those.
__device__ __forceinline__ int dz_exp(uint32_t half) { return pr::scale_exp(half) - 1; }

// The largest finite |W|, |X| and half the bound of |dZ| of a piece's rows, by blocks.
__global__ void __launch_bounds__(1024) ffn_max_kernel(FfnArgs a) {
  __shared__ uint32_t part[16];
  uint32_t m = 0;
  int bid = (int)blockIdx.x, kind = 2;  // the most work first
  while (kind > 0 && bid >= a.max_blocks[kind]) bid -= a.max_blocks[kind--];
  const int blocks = a.max_blocks[kind];
  constexpr int U = 4;  // loads of each operand under way
  if (kind == 0) {
    const int64_t n = a.D * 2 * a.F, step = (int64_t)blocks * 4096;
    for (int64_t i0 = ((int64_t)bid * 1024 + threadIdx.x) * 4; i0 < n; i0 += U * step) {
      f32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * step;
        x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (i + 4 <= n) {
          x[u] = *reinterpret_cast<const f32x4u*>(a.W + i);
        } else {
          for (int e = 0; e < 4; ++e)
            if (i + e < n) x[u][e] = a.W[i + e];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[u][e]));
    }
  } else {
    // items of 256 rows of a column, a wave each: item t is chunk t % chunks of column
    // t / chunks, kept up by additions
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunks = (int)((a.R + 255) / 256), step = blocks * 16;
    const int64_t cols = kind == 1 ? a.D : a.F;
    const int step_cols = step / chunks, step_chunks = step % chunks;
    int64_t col = (bid * 16 + wave) / chunks;
    int chunk = (bid * 16 + wave) % chunks;
    // behind the last rows the last four again, so that no load stands behind a test of its
    // own and is waited for (a piece of fewer than four rows: one row a lane)
    auto get = [&](const float* p, int n) {
      if (a.R >= 4) return f32x4(*reinterpret_cast<const f32x4u*>(p + (n + 4 <= a.R ? n : a.R - 4)));
      const float x = p[n < a.R ? n : 0];
      return f32x4{x, x, x, x};
    };
    while (col < cols) {
      f32x4 x[U], y[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int n = chunk * 256 + (a.R >= 4 ? 4 * lane : lane);
        const int64_t at = a.row0 + a.N * (col < cols ? col : cols - 1);
        x[u] = get((kind == 1 ? a.X : a.Z) + at, n);
        if (kind == 2) {
          y[u] = get(a.Z + a.N * a.F + at, n);
          z[u] = get(a.dH + at, n);
        }
        col += step_cols;
        chunk += step_chunks;
        if (chunk >= chunks) {
          chunk -= chunks;
          ++col;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (kind == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[u][e]));
          continue;
        }
        // (told apart for every four: for each value 0.8 us longer in 1021 x 1365, for all 16
        // they need more registers than two blocks on a CU have)
        with_act(a.act, [&](auto act) {
#pragma unroll
          for (int e = 0; e < 4; ++e) m = max(m, half_grad_bound(act, x[u][e], y[u][e], z[u][e]));
        });
      }
    }
  }
  m = pr::wave_max(m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) m = max(m, part[w]);
  a.max_part[kMaxAt[kind] + bid] = m;
}

// Of all the blocks that looked at operand `kind`, in every lane.
__device__ __forceinline__ uint32_t max_of(const FfnArgs& a, int kind) {
  uint32_t m = 0;
  for (int i = threadIdx.x & 63; i < a.max_blocks[kind]; i += 64) m = max(m, a.max_part[kMaxAt[kind] + i]);
  return pr::wave_max(m);
}

// What the products of the backward read, packed; a wave for
//   - a step of 16 hidden features of dZ and z_blocks blocks of 32 rows, with its column
//     sums where they are wanted (the first z_waves waves),
//   - a fragment of W^T, of X.
__global__ void __launch_bounds__(256) ffn_pack_kernel(FfnArgs a, int64_t z_waves, int64_t w_frags, int64_t x_frags) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int64_t blocks = (a.R + 31) / 32;
  int64_t f = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (f == 0) {  // for the products
    const FfnScales s{max_of(a, 0), max_of(a, 1), max_of(a, 2)};
    if (lane == 0) *a.scales = s;
  }
  if (f < z_waves) {
    const int64_t groups = (blocks + a.z_blocks - 1) / a.z_blocks, grp = f % groups;
    const int step = (int)(f / groups);
    const int64_t f0 = (int64_t)step * 16 + 8 * h;
    const float s = pr::exp2i(dz_exp(max_of(a, 2)));
    float sg[8] = {}, su[8] = {};
    for (int64_t b = grp * a.z_blocks; b < (grp + 1) * a.z_blocks && b < blocks; ++b) {
      const int64_t n = b * 32 + r;
      float zg[8], zu[8], dh[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = n < a.R && f0 + e < a.F;
        const int64_t at = a.row0 + n + a.N * (f0 + e);
        zg[e] = in ? a.Z[at] : 0.f;
        zu[e] = in ? a.Z[a.N * a.F + at] : 0.f;
        dh[e] = in ? a.dH[at] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float dg, du;
        grads_of(a, zg[e], zu[e], dh[e], dg, du);
        sg[e] += dg;
        su[e] += du;
        zg[e] = dg * s;
        zu[e] = du * s;
      }
      const int at = 4 * (step >> 1) + (step & 1);  // the gate's step of the packed columns; the up's is two on
      pr::put_frag(a.zp, b, 2 * a.steps_f, at, zg);
      pr::put_frag(a.zp, b, 2 * a.steps_f, at + 2, zu);
    }
    if (!a.db_part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sg[e] += __shfl_xor(sg[e], o, 64);
        su[e] += __shfl_xor(su[e], o, 64);
      }
      if (r == 0 && f0 + e < a.F) {
        a.db_part[grp * 2 * a.F + f0 + e] = sg[e];
        a.db_part[grp * 2 * a.F + a.F + f0 + e] = su[e];
      }
    }
    return;
  }
  f -= z_waves;
  float x[8];
  if (f < w_frags) {
    const int64_t col = column_of(f / a.steps_d * 32 + r, a.F);
    const int step = (int)(f % a.steps_d);
    const int64_t d0 = step * 16 + 8 * h;
    const float* p = a.W + col * a.D + d0;
    if (col >= 0 && d0 + 8 <= a.D) {
      const f32x4 u = *reinterpret_cast<const f32x4u*>(p), w = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = u[e];
        x[4 + e] = w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = col >= 0 && d0 + e < a.D ? p[e] : 0.f;
    }
    const float s = pr::exp2i(pr::scale_exp(max_of(a, 0)));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= s;
    pr::put_frag(a.wp, f / a.steps_d, a.steps_d, step, x);
    return;
  }
  f -= w_frags;
  if (f >= x_frags) return;
  // neighbouring waves take neighbouring row blocks: their reads run along a column
  const int64_t n = f % blocks * 32 + r;
  const int step = (int)(f / blocks);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t d = step * 16 + 8 * h + e;
    x[e] = n < a.R && d < a.D ? a.X[a.row0 + n + a.N * d] : 0.f;
  }
  const float s = pr::exp2i(pr::scale_exp(max_of(a, 1)));
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= s;
  pr::put_frag(a.xp, f % blocks, a.steps_d, step, x);
}

struct FfnOut {
  float* p;
  int64_t ld;
  float* part;  // split sums [splits][M][N], or null
  int accumulate;
};
// COLS: row m of the product is column_of(m) of the output.
template <bool COLS>
__device__ __forceinline__ int scale_out(const FfnArgs& a) {
  return -dz_exp(a.scales->z) - pr::scale_exp(COLS ? a.scales->x : a.scales->w);
}

// A product of the backward as blocks [tile][split].
struct FfnProduct {
  pr::GemmArgs g;
  FfnOut o;
  int tiles, splits;
};

// dX (A: W across its rows, B: dZ), COLS false, and dW (A: dZ, B: X, both across
// their rows), COLS true.
template <class T, bool TA, bool TB, bool COLS>
__device__ __forceinline__ void ffn_product(const FfnProduct& p, const FfnArgs& a, int bid, char* lds) {
  const pr::GemmArgs& g = p.g;
  const FfnOut& o = p.o;
  int tm, tn;
  const int split = bid / p.tiles;
  pr::tile_of(bid % p.tiles, (g.M + T::TM - 1) / T::TM, (g.N + T::TN - 1) / T::TN, tm, tn);
  const int t0 = split * g.steps_per_split, t1 = min(g.steps, t0 + g.steps_per_split);
  pr::AccOf<T::MI> acc;
  pr::gemm_tile<TA, TB, T>(g, tm, tn, t0, t1, lds, acc);
  if (o.part) {
    pr::put_tile<false, T>(acc, tm, tn, g.M, g.N, o.part + (int64_t)split * g.M * g.N, g.N, [](float x) { return x; });
    return;
  }
  const int eo = scale_out<COLS>(a);
  auto value = [&](float x) { return pr::times_exp2(x, eo); };
  if constexpr (!COLS) {
    pr::put_tile<false, T>(acc, tm, tn, g.M, g.N, o.p, o.ld, value);
  } else {
    // blocks of 32 packed columns lie together in the output: the even ones from its
    // start on, the odd ones from column F on
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < T::J; ++j) {
      const int n = tn * T::TN + T::column(j);
      if (n >= g.N) continue;
#pragma unroll
      for (int i = 0; i < T::MI; ++i) {
        const int64_t blk = (tm * T::TM + T::row0()) / 32 + i;
        const int64_t f = (blk >> 1) * 32 + 4 * (lane >> 5), left = a.F - f;
        float* q = o.p + n + o.ld * (f + (blk & 1) * a.F);
        auto row = [](int e) { return 8 * (e / 4) + e % 4; };
        if (!o.accumulate) {
          if (left >= 32) {
#pragma unroll
            for (int e = 0; e < 16; ++e) q[o.ld * row(e)] = value(acc.x[i][j][e]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (row(e) < left) q[o.ld * row(e)] = value(acc.x[i][j][e]);
          }
          continue;
        }
        float old[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = row(e) < left ? q[o.ld * row(e)] : 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (row(e) < left) q[o.ld * row(e)] = old[e] + value(acc.x[i][j][e]);
      }
    }
  }
}

// Both products, the one of the longer blocks first, so that the shorter ones fill what is
// left (3822 x 652 -> 1121 in small tiles: 30 us of 180), and db (+)= the sums of the
// groups of rows, in order, in the blocks behind them.
template <class T>
__global__ void __launch_bounds__(T::NT, 2) ffn_grads_kernel(FfnArgs a, FfnProduct x, FfnProduct w, float* db, int add) {
  __shared__ __align__(16) char lds[T::kLds];
  const int nx = x.tiles * x.splits, nw = w.tiles * w.splits;
  const bool w_first = w.g.steps_per_split > x.g.steps_per_split;
  int bid = (int)blockIdx.x;
  if (bid < nx + nw) {
    if (w_first ? bid >= nw : bid < nx) ffn_product<T, true, false, false>(x, a, w_first ? bid - nw : bid, lds);
    else ffn_product<T, true, true, true>(w, a, w_first ? bid : bid - nx, lds);
    return;
  }
  bid -= nx + nw;
  const int64_t v = (int64_t)bid * T::NT + threadIdx.x, blocks = (a.R + 31) / 32;
  if (v >= 2 * a.F) return;
  float s = 0.f;
#pragma unroll 16
  for (int64_t q = 0; q < (blocks + a.z_blocks - 1) / a.z_blocks; ++q) s += a.db_part[q * 2 * a.F + v];
  db[v] = add ? db[v] + s : s;
}

// A row's 256 sums of a product that was split; block: [row][256 columns].
template <bool COLS>
__device__ __forceinline__ void ffn_reduce(const FfnProduct& p, const FfnArgs& a, int block) {
  const int chunks = (p.g.N + 255) / 256, m = block / chunks, n = block % chunks * 256 + threadIdx.x;
  const int64_t to = COLS ? column_of(m, a.F) : m, total = (int64_t)p.g.M * p.g.N;
  if (to < 0 || n >= p.g.N) return;
  const float* from = p.o.part + (int64_t)m * p.g.N + n;
  float x = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) x += from[s * total];
  float* q = p.o.p + n + p.o.ld * to;
  x = pr::times_exp2(x, scale_out<COLS>(a));
  *q = p.o.accumulate ? *q + x : x;
}
// The products that were split, the x_blocks blocks of the first before the second's.
__global__ void __launch_bounds__(256) ffn_reduce_kernel(FfnArgs a, FfnProduct x, FfnProduct w, int x_blocks) {
  const int bid = (int)blockIdx.x;
  if (bid < x_blocks) ffn_reduce<false>(x, a, bid);
  else ffn_reduce<true>(w, a, bid - x_blocks);
}

template <class T>
int64_t tiles_of(int64_t M, int64_t N) {
  return (M + T::TM - 1) / T::TM * ((N + T::TN - 1) / T::TN);
}
int64_t pad32(int64_t n) { return (n + 31) / 32 * 32; }

struct Places {
  size_t at = 0;
  size_t place(size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
};

int check_shape(int64_t N, int64_t D, int64_t F, int act, const char* who) {
  CNHIP_REQUIRE(N > 0 && D > 0 && F > 0, "%s: bad shape batch=%lld in_features=%lld hidden=%lld", who, (long long)N,
                (long long)D, (long long)F);
  CNHIP_REQUIRE(act >= CNHIP_GATE_SILU && act <= CNHIP_GATE_RELU, "%s: bad activation %d", who, act);
  // (a grid has fewer than 2^32 threads; the packing has 32 for a row or a column of W)
  CNHIP_REQUIRE(N < ((int64_t)1 << 26) && D < ((int64_t)1 << 22) && F < ((int64_t)1 << 25), "%s: too large", who);
  return CNHIP_OK;
}

struct Job {
  int64_t M, N;
  int steps;
};
struct Plan {
  int per[2] = {};  // steps of a block of each product
  double us = 0;
};
// What a step costs a block that has the chip's caches to itself and one among as many as
// run at a time, us; steps that a block's beginning and end take, where it stores split
// sums and where it does not; bytes of split sums a us.
struct Rates {
  double light, full, ends_split, ends, bytes;
  int slots;  // blocks at a time
};
// Read off the kernels' times for 13 shapes from 300 x 256 -> 512 to 16384 x 128 -> 256 and 2048 x
// 1024 -> 4096, which these give again to some 15%.
template <class T>
constexpr Rates kRates = T::G == 2   ? Rates{0.28, 0.42, 18, 18, 6e6, 256}
                         : T::WN == 2 ? Rates{0.75, 1.2, 7, 17, 8e6, 512}
                                      : Rates{1.45, 1.45, 8, 8, 9e6, 256};
int even(int64_t n) { return (int)((n + 1) / 2 * 2); }
// The splits where all the products of a launch are done soonest.
template <class T>
Plan plan_of(const Job* jobs, int n) {
  constexpr Rates r = kRates<T>;
  int longest = 2;
  for (int i = 0; i < n; ++i) longest = jobs[i].steps > longest ? jobs[i].steps : longest;
  Plan best;
  for (int parts = 1; parts <= 64; ++parts) {
    const int most = even((longest + parts - 1) / parts);
    if (parts > 1 && most < 6) break;
    Plan p;
    double moved = 0, work = 0, blocks = 0, block = 0, shortest = 0;
    for (int i = 0; i < n; ++i) {
      const int steps = jobs[i].steps, alike = (steps + most - 1) / most;
      p.per[i] = even((steps + alike - 1) / alike);
      const int splits = (steps + p.per[i] - 1) / p.per[i];
      const double b = (double)(tiles_of<T>(jobs[i].M, jobs[i].N) * splits), own = p.per[i] + (splits > 1 ? r.ends_split : r.ends);
      blocks += b;
      work += b * own;
      block = own > block ? own : block;
      shortest = i == 0 || own < shortest ? own : shortest;
      if (splits > 1) moved += 8.0 * splits * (double)jobs[i].M * (double)jobs[i].N;
    }
    const double rounds = work / block / r.slots;
    double step = blocks <= 256 ? r.light : r.full * std::ceil(rounds);
    if (T::G == 2 && (n == 2 || blocks <= r.slots)) {
      // blocks of two lengths fill a round that one of them leaves half empty
      step = r.full * (rounds + (blocks > r.slots ? 0.5 * shortest / block : 0.0));
    }
    p.us = 3 + block * (step > r.light ? step : r.light) + (moved > 0 ? 4 + moved / r.bytes : 0);
    if (best.us == 0 || p.us < best.us) best = p;
    if (blocks > 4 * r.slots) break;  // more of them win nothing
  }
  return best;
}
// f(a tile): Small's or T
template <class T, class F>
void with_tile(bool small, F&& f) {
  if (small) f(Small{});
  else f(T{});
}

int run_forward(FfnArgs& a, hipStream_t st, const char* who) {
  const int64_t N = a.N, D = a.D, F = a.F, Fp = pad32(F);
  if (few_rows(N, D, F)) {
    const dim3 grid((unsigned)((F + 7) / 8), (unsigned)((N + kFewBlock - 1) / kFewBlock)), threads(512);
    if (N <= 16) hipLaunchKernelGGL(ffn_few_kernel<1>, grid, threads, 0, st, a);
    else if (N <= 32) hipLaunchKernelGGL(ffn_few_kernel<2>, grid, threads, 0, st, a);
    else if (N <= 64) hipLaunchKernelGGL(ffn_few_kernel<4>, grid, threads, 0, st, a);
    else hipLaunchKernelGGL(ffn_few_kernel<8>, grid, threads, 0, st, a);
    return check_launch(who);
  }
  a.steps_d = (int)(pad32(D) / 16);
  CNHIP_REQUIRE(tiles_of<Small>(2 * Fp, N) < ((int64_t)1 << 23), "%s: too large", who);
  Places w;
  const size_t o_x = w.place((size_t)(pad32(N) * pad32(D)) * 4), o_w = w.place((size_t)(2 * Fp * pad32(D)) * 4),
               o_xe = w.place((size_t)N * 4), o_we = w.place((size_t)(2 * Fp / 32) * 4);
  const Job job{2 * Fp, N, a.steps_d};
  // (a row of the grid for every feature joins the splits)
  const Plan half = plan_of<Half>(&job, 1), few = plan_of<Small>(&job, 1);
  const bool small = few.us < half.us;
  const int per = F < 65536 ? (small ? few : half).per[0] : a.steps_d, splits = (a.steps_d + per - 1) / per;
  const size_t o_part = w.place(splits > 1 ? (size_t)(splits * 2 * Fp * N) * 4 : 0);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, w.at, &ws, who));
  char* base = static_cast<char*>(ws);
  a.xp = base + o_x;
  a.wp = base + o_w;
  a.xe = reinterpret_cast<int*>(base + o_xe);
  a.we = reinterpret_cast<int*>(base + o_we);
  hipLaunchKernelGGL(ffn_pack_own_kernel, dim3((unsigned)(2 * Fp / 32 + pad32(N) / 32)), dim3(1024), 0, st, a,
                     (int)(2 * Fp / 32));
  CNHIP_TRY(check_launch(who));
  const pr::GemmArgs g{pr::Packed{a.wp, (int)(2 * Fp / 32), a.steps_d}, pr::Packed{a.xp, (int)(pad32(N) / 32), a.steps_d},
                       (int)(2 * Fp), (int)N, a.steps_d, per, a.steps_d / 2};
  float* part = splits > 1 ? reinterpret_cast<float*>(base + o_part) : nullptr;
  with_tile<Half>(small, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(ffn_forward_kernel<T>, dim3((unsigned)tiles_of<T>(2 * Fp, N), (unsigned)splits), dim3(T::NT), 0, st, g,
                       a, part);
  });
  CNHIP_TRY(check_launch(who));
  if (!part) return CNHIP_OK;
  hipLaunchKernelGGL(ffn_join_kernel, dim3((unsigned)((N + 255) / 256), (unsigned)F), dim3(256), 0, st, a, part, 2 * Fp,
                     splits);
  return check_launch(who);
}

// Few rows: dZ, and the Linear's backward over it.  This way and packed, both with the
// forward, us: 512 -> 2048 65 rows 40 and 44, 128 rows 43 and 44, 256 rows 64 and 58; 1024 ->
// 4096 64 rows 67 and 82, 128 rows 103 and 106, 256 rows 147 and 132; 1024 -> 1024 96 rows 47
// and 51; 256 -> 512 256 rows 31.5 and 36; 2048 -> 8192 64 rows 204 and 251.
bool few_rows_back(int64_t N, int64_t D, int64_t F) {
  return N <= 96 || (N <= 256 && (double)N * (double)D * (double)F <= 1.5e8);
}

int run_backward_few(FfnArgs& a, float* dX, float* dW, float* db, int accumulate, hipStream_t st, const char* who) {
  void* dZ = nullptr;
  const int64_t n = a.N * a.F;
  CNHIP_REQUIRE((n + 1023) / 1024 < ((int64_t)1 << 24), "%s: too large", who);
  CNHIP_TRY(scratch(st, kScratchLayer, (size_t)(2 * n) * sizeof(float), &dZ, who));
  hipLaunchKernelGGL(ffn_dz_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, a, static_cast<float*>(dZ));
  CNHIP_TRY(check_launch(who));
  return cnhip_linear_backward(a.X, a.W, static_cast<float*>(dZ), dW, db, dX, a.N, a.D, 2 * a.F, 1, accumulate, st);
}

int run_backward(FfnArgs& a, float* dX, float* dW, float* db, int accumulate, hipStream_t st, const char* who) {
  const int64_t N = a.N, D = a.D, F = a.F, Fp = pad32(F), Dp = pad32(D);
  a.steps_d = (int)(Dp / 16);
  a.steps_f = (int)(Fp / 16);
  // Rows of a piece: 2^27 values of dZ (half a GiB packed), but 1024 rows at least, so
  // that dW is read and written once in 1024 rows at most.
  const int64_t most = ((int64_t)1 << 27) / (2 * Fp);
  int64_t R = most < 1024 ? 1024 : most / 256 * 256;
  if (R > N) R = N;
  const int64_t Rp = pad32(R);
  const Job jobs[2] = {{D, R, 2 * a.steps_f}, {2 * Fp, D, (int)(Rp / 16)}};
  const Plan whole = plan_of<Whole>(jobs, 2), few = plan_of<Small>(jobs, 2);
  const bool small = few.us < whole.us;
  const Plan& plan = small ? few : whole;
  auto parts = [&](int i) {
    const int64_t splits = (jobs[i].steps + plan.per[i] - 1) / plan.per[i];
    return splits > 1 ? (size_t)(splits * jobs[i].M * jobs[i].N) * 4 : 0;
  };
  CNHIP_REQUIRE(tiles_of<Small>(D, R) * ((2 * a.steps_f + plan.per[0] - 1) / plan.per[0]) +
                        tiles_of<Small>(2 * Fp, D) * ((Rp / 16 + plan.per[1] - 1) / plan.per[1]) <
                    ((int64_t)1 << 22),
                "%s: too large", who);
  // blocks of 32 rows of dZ a wave: as many as leave 4096 waves, so that a wave that has
  // several keeps its loads going
  a.z_blocks = 8;
  while (a.z_blocks > 1 && Rp / 32 / a.z_blocks * a.steps_f < 4096) a.z_blocks /= 2;
  Places w;
  const size_t o_max = w.place(kMaxParts * 4 + sizeof(FfnScales)), o_x = w.place((size_t)(Rp * Dp) * 4),
               o_w = w.place((size_t)(2 * Fp * Dp) * 4), o_z = w.place((size_t)(Rp * 2 * Fp) * 4),
               o_db = w.place(db ? (size_t)((Rp / 32 + a.z_blocks - 1) / a.z_blocks * 2 * F) * 4 : 0),
               o_px = w.place(parts(0)), o_pw = w.place(parts(1));
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, w.at, &ws, who));
  char* base = static_cast<char*>(ws);
  a.max_part = reinterpret_cast<uint32_t*>(base + o_max);
  a.scales = reinterpret_cast<FfnScales*>(base + o_max + kMaxParts * 4);
  a.xp = base + o_x;
  a.wp = base + o_w;
  a.zp = base + o_z;
  a.db_part = db ? reinterpret_cast<float*>(base + o_db) : nullptr;
  const pr::Packed pw_{a.wp, (int)(2 * Fp / 32), a.steps_d};
  auto product = [&](const pr::Packed& A, const pr::Packed& B, int64_t M, int64_t Nn, int steps, int per, float* p,
                     int64_t ld, float* part, int add) {
    const int splits = (steps + per - 1) / per;
    return FfnProduct{pr::GemmArgs{A, B, (int)M, (int)Nn, steps, per, steps / 2},
                      FfnOut{p, ld, splits > 1 ? part : nullptr, add},
                      (int)(small ? tiles_of<Small>(M, Nn) : tiles_of<Whole>(M, Nn)), splits};
  };
  for (int64_t r0 = 0; r0 < N; r0 += R) {
    a.row0 = r0;
    a.R = N - r0 < R ? N - r0 : R;
    const int rb = (int)((a.R + 31) / 32);
    // with loads for every thread, as far as there are any
    const int64_t wanted[3] = {r0 ? a.max_blocks[0] : 2 * D * F / 16384, D * ((a.R + 255) / 256) / 64,
                               F * ((a.R + 255) / 256) / 32};
    for (int k = 0; k < 3; ++k)
      a.max_blocks[k] = (int)(wanted[k] < 1 ? 1 : wanted[k] > kMaxBlocks[k] ? kMaxBlocks[k] : wanted[k]);
    hipLaunchKernelGGL(ffn_max_kernel, dim3((unsigned)(a.max_blocks[0] + a.max_blocks[1] + a.max_blocks[2])), dim3(1024), 0,
                       st, a);
    CNHIP_TRY(check_launch(who));
    const int64_t zw = (int64_t)((rb + a.z_blocks - 1) / a.z_blocks) * a.steps_f, wf = r0 ? 0 : 2 * Fp / 32 * a.steps_d,
                  xf = (int64_t)rb * a.steps_d;
    CNHIP_REQUIRE(zw + wf + xf < ((int64_t)1 << 25), "%s: too large", who);
    hipLaunchKernelGGL(ffn_pack_kernel, dim3((unsigned)((zw + wf + xf + 3) / 4)), dim3(256), 0, st, a, zw, wf, xf);
    CNHIP_TRY(check_launch(who));
    const int add = accumulate || r0 > 0;
    const pr::Packed px_{a.xp, rb, a.steps_d}, pz_{a.zp, rb, 2 * a.steps_f};
    const FfnProduct x = product(pw_, pz_, D, a.R, 2 * a.steps_f, plan.per[0], dX + r0, N, reinterpret_cast<float*>(base + o_px), 0),
                     y = product(pz_, px_, 2 * Fp, D, 2 * rb, plan.per[1], dW, D, reinterpret_cast<float*>(base + o_pw), add);
    with_tile<Whole>(small, [&](auto t) {
      using T = decltype(t);
      const int64_t blocks = (int64_t)x.tiles * x.splits + (int64_t)y.tiles * y.splits + (db ? (2 * F + T::NT - 1) / T::NT : 0);
      hipLaunchKernelGGL(ffn_grads_kernel<T>, dim3((unsigned)blocks), dim3(T::NT), 0, st, a, x, y, db, add);
    });
    CNHIP_TRY(check_launch(who));
    if (!x.o.part && !y.o.part) continue;
    auto reduce_blocks = [](const FfnProduct& q) { return q.o.part ? (int64_t)q.g.M * ((q.g.N + 255) / 256) : 0; };
    const int64_t xb = reduce_blocks(x), wb = reduce_blocks(y);
    CNHIP_REQUIRE(xb + wb < ((int64_t)1 << 24), "%s: too large", who);
    hipLaunchKernelGGL(ffn_reduce_kernel, dim3((unsigned)(xb + wb)), dim3(256), 0, st, a, x, y, (int)xb);
    CNHIP_TRY(check_launch(who));
  }
  return CNHIP_OK;
}

}  // namespace
}  // namespace cnhip

extern "C" {

int cnhip_gated_ffn_forward(const float* X, const float* W, const float* b, float* H, float* Z, int64_t batch,
                            int64_t in_features, int64_t hidden, int act, cnhip_stream_t stream) {
  const char* who = "cnhip_gated_ffn_forward";
  CNHIP_TRY(cnhip::check_shape(batch, in_features, hidden, act, who));
  CNHIP_REQUIRE(X && W && H, "%s: NULL pointer", who);
  cnhip::FfnArgs a{};
  a.X = X;
  a.W = W;
  a.b = b;
  a.H = H;
  a.Zout = Z;
  a.N = batch;
  a.D = in_features;
  a.F = hidden;
  a.act = act;
  return cnhip::run_forward(a, cnhip::as_stream(stream), who);
}

int cnhip_gated_ffn_backward(const float* X, const float* W, const float* Z, const float* dH, float* dX, float* dW,
                             float* db, int64_t batch, int64_t in_features, int64_t hidden, int act, int accumulate,
                             cnhip_stream_t stream) {
  const char* who = "cnhip_gated_ffn_backward";
  CNHIP_TRY(cnhip::check_shape(batch, in_features, hidden, act, who));
  CNHIP_REQUIRE(X && W && Z && dH && dX && dW, "%s: NULL pointer", who);
  CNHIP_REQUIRE(accumulate == 0 || accumulate == 1, "%s: accumulate must be 0 or 1", who);
  cnhip::FfnArgs a{};
  a.X = X;
  a.W = W;
  a.Z = Z;
  a.dH = dH;
  a.N = batch;
  a.D = in_features;
  a.F = hidden;
  a.act = act;
  const hipStream_t st = cnhip::as_stream(stream);
  return cnhip::few_rows_back(batch, in_features, hidden) ? cnhip::run_backward_few(a, dX, dW, db, accumulate, st, who)
                                                          : cnhip::run_backward(a, dX, dW, db, accumulate, st, who);
}

}  // extern "C"
