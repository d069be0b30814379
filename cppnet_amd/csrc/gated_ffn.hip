// A gated feed-forward layer: two projections, an activation of the first and
// the product with the second, in one call, and its backward pass.
//
//   Z = X W + b, gate = Z[:, :F], up = Z[:, F:],  H = act(gate) up
// backward:
//   dgate = dH up act'(gate), dup = dH act(gate), dZ = [dgate dup],
//   dX = dZ W^T,  dW (+)= X^T dZ,  db (+)= column sums of dZ
//
// The products run on the fp16 matrix cores over operands packed as pairs
// (mfma_pair.hpp).  W's columns are packed in blocks of 32, a gate's and then its
// up's, so one wave's accumulators hold both values of an element and the
// activation and the product are done where the sums are.  dZ is packed in the
// same order of columns straight from Z and dH, and serves both products of the
// backward, once along its columns and once along its rows.
#include <hip/hip_runtime.h>

#include "act_math.hpp"
#include "common.hpp"
#include "mfma_pair.hpp"

namespace cnhip {
namespace {

using pr::f32x16;
using pr::f32x4;
using pr::f32x4u;

// Largest finite values, as bits: of W, and of a piece's X and dZ.
struct FfnScales {
  uint32_t x, z;
};

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
  uint32_t* w_max;
  FfnScales* scales;   // the piece's
  float* db_part;      // [ceil(R / 256)][2 F], or null
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
// act(z)
__device__ __forceinline__ float gate_f(int act, float z) {
  if (act == CNHIP_GATE_GELU) return gelu_f(z);
  if (act == CNHIP_GATE_RELU) return relu_f(z);
  float on, off;
  sigmoid_parts(z, on, off);
  return act == CNHIP_GATE_SILU ? z * on : on;
}
// act(z) and act'(z)
__device__ __forceinline__ void gate_both(int act, float z, float& y, float& d) {
  if (act == CNHIP_GATE_GELU) {
    float e;  // exp(-z^2 / 2)
    const float cdf = ncdf_f(z, fabsf(z) * 0.70710678118654752440f, &e);
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

// ------------------------------------------------------------------ forward
// X and W^T packed, every row of X and every 32 rows of W^T with an exponent of
// their own: a block of eight waves for 32 rows, which reads them twice (the
// second time from the L2).
__global__ void __launch_bounds__(512) ffn_pack_own_kernel(FfnArgs a, int w_blocks) {
  __shared__ uint32_t part[8][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const bool w = (int)blockIdx.x < w_blocks;
  const int64_t blk = w ? blockIdx.x : (int64_t)blockIdx.x - w_blocks, row = blk * 32 + r;
  const int64_t col = w ? column_of(row, a.F) : 0;
  const bool in = w ? col >= 0 : row < a.N;
  auto load = [&](int step, float (&x)[8]) {
    const int64_t d0 = step * 16 + 8 * h;
    if (w) {
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
  for (int s0 = wave; s0 < a.steps_d; s0 += 32) {
    float x[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (s0 + 8 * u < a.steps_d) load(s0 + 8 * u, x[u]);
      else
        for (int e = 0; e < 8; ++e) x[u][e] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, pr::finite_bits(x[u][e]));
  }
  if (w) m = pr::wave_max(m);
  else m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  if (lane < 32) part[wave][lane] = m;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 8; ++q) m = max(m, part[q][r]);
  const int exp = pr::scale_exp(m);
  const float f = pr::exp2i(exp);
  if (wave == 0 && lane < 32) {
    if (!w && in) a.xe[row] = exp;
    if (w && lane == 0) a.we[blk] = exp;
  }
  for (int step = wave; step < a.steps_d; step += 8) {
    float x[8];
    load(step, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f;
    pr::put_frag(w ? a.wp : a.xp, blk, a.steps_d, step, x);
  }
}

// A: W^T (M: packed columns), B: X (N: rows); H and, where it is kept, Z.
__global__ void __launch_bounds__(pr::GNT, 2) ffn_forward_kernel(pr::GemmArgs g, FfnArgs a) {
  __shared__ __align__(16) char lds[pr::kGemmLds];
  int tm, tn;
  pr::tile_of((int)blockIdx.x, (g.M + pr::TM - 1) / pr::TM, (g.N + pr::TN - 1) / pr::TN, tm, tn);
  pr::Acc acc;
  pr::gemm_tile<false, false>(g, tm, tn, 0, g.steps, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int block0 = tm * (pr::TM / 32) + (wave >> 2) * 4;  // the wave's first of 32 packed columns: a gate's
  int64_t n[2];
  int ex[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    n[j] = (int64_t)tn * pr::TN + (wave & 3) * 64 + 32 * j + (lane & 31);
    ex[j] = a.xe[n[j] < a.N ? n[j] : a.N - 1];
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    if (block0 + i >= g.M / 32) break;
    const int eg = a.we[block0 + i], eu = a.we[block0 + i + 1];
    const int64_t f0 = (int64_t)(block0 + i) * 16 + 4 * (lane >> 5);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t f = f0 + 8 * (e / 4) + e % 4;
      if (f >= a.F) continue;
      const float bg = a.b ? a.b[f] : 0.f, bu = a.b ? a.b[a.F + f] : 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (n[j] >= a.N) continue;
        const float gate = pr::times_exp2(acc.x[i][j][e], -ex[j] - eg) + bg;
        const float up = pr::times_exp2(acc.x[i + 1][j][e], -ex[j] - eu) + bu;
        if (a.Zout) {
          a.Zout[n[j] + a.N * f] = gate;
          a.Zout[n[j] + a.N * (a.F + f)] = up;
        }
        a.H[n[j] + a.N * f] = gate_f(a.act, gate) * up;
      }
    }
  }
}

// Few rows: W is read once and each value used for a handful of products, so the
// fp32 matrix cores keep up with memory and nothing is packed.  A block takes 8
// hidden features (16 columns of W, the rows of the 16 x 16 tiles); its eight
// waves share out D and meet in LDS.
constexpr int kFewRows = 64;
template <int NB>
__global__ void __launch_bounds__(512) ffn_few_kernel(FfnArgs a) {
  __shared__ float part[8][16][16 * NB + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int64_t f0 = (int64_t)blockIdx.x * 8, f = f0 + (r & 7);
  const float* w = a.W + ((r >> 3) * a.F + (f < a.F ? f : a.F - 1)) * a.D;
  const int N = (int)a.N;
  f32x4 acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = NB > 2 ? 2 : 4;  // steps of 16 features under way
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
          xv[u][j][e] = d + e < a.D && 16 * j + r < N ? a.X[16 * j + r + a.N * (d + e)] : 0.f;
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
    if (a.Zout) {
      a.Zout[n + a.N * (f0 + k)] = gate;
      a.Zout[n + a.N * (a.F + f0 + k)] = up;
    }
    a.H[n + a.N * (f0 + k)] = gate_f(a.act, gate) * up;
  }
}

// ----------------------------------------------------------------- backward
__device__ __forceinline__ void grads_of(const FfnArgs& a, float gate, float up, float dh, float& dg, float& du) {
  float y, d;
  gate_both(a.act, gate, y, d);
  dg = dh * up * d;
  du = dh * y;
}

// The largest finite |W| (the first w_blocks blocks, with the first piece), |X| (x_blocks)
// and |dZ| of a piece's rows.
__global__ void __launch_bounds__(256) ffn_max_kernel(FfnArgs a, int w_blocks, int x_blocks) {
  uint32_t m = 0;
  uint32_t* to;
  int bid = (int)blockIdx.x;
  const int64_t chunks = (a.R + 1023) / 1024;  // of rows
  if (bid < w_blocks) {
    to = a.w_max;
    const int64_t n = a.D * 2 * a.F, step = (int64_t)w_blocks * 1024;
    for (int64_t i = ((int64_t)bid * 256 + threadIdx.x) * 4; i < n; i += step) {
      if (i + 4 <= n) {
        const f32x4 x = *reinterpret_cast<const f32x4u*>(a.W + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[e]));
      } else {
        for (int64_t e = i; e < n; ++e) m = max(m, pr::finite_bits(a.W[e]));
      }
    }
  } else if ((bid -= w_blocks) < x_blocks) {
    to = &a.scales->x;
    for (int64_t t = bid; t < a.D * chunks; t += x_blocks) {
      const int64_t n = t % chunks * 1024 + 4 * threadIdx.x;
      const float* p = a.X + a.row0 + n + a.N * (t / chunks);
      if (n + 4 <= a.R) {
        const f32x4 x = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[e]));
      } else {
        for (int e = 0; n + e < a.R; ++e) m = max(m, pr::finite_bits(p[e]));
      }
    }
  } else {
    bid -= x_blocks;
    to = &a.scales->z;
    const int z_blocks = (int)gridDim.x - w_blocks - x_blocks;
    for (int64_t t = bid; t < a.F * chunks; t += z_blocks) {
      const int64_t n = t % chunks * 1024 + 4 * threadIdx.x, at = a.row0 + n + a.N * (t / chunks);
      f32x4 zg = {0.f, 0.f, 0.f, 0.f}, zu = zg, dh = zg;
      if (n + 4 <= a.R) {
        zg = *reinterpret_cast<const f32x4u*>(a.Z + at);
        zu = *reinterpret_cast<const f32x4u*>(a.Z + a.N * a.F + at);
        dh = *reinterpret_cast<const f32x4u*>(a.dH + at);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (n + e >= a.R) continue;
          zg[e] = a.Z[at + e];
          zu[e] = a.Z[a.N * a.F + at + e];
          dh[e] = a.dH[at + e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float dg, du;
        grads_of(a, zg[e], zu[e], dh[e], dg, du);
        m = max(m, max(pr::finite_bits(dg), pr::finite_bits(du)));
      }
    }
  }
  __shared__ uint32_t part[4];
  m = pr::wave_max(m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x) return;
  m = max(max(part[0], part[1]), max(part[2], part[3]));
  if (m) atomicMax(to, m);  // a maximum is the same in any order
}

// W^T (with the first piece) and the piece's rows of X packed, a wave per fragment.
__global__ void __launch_bounds__(256) ffn_pack_kernel(FfnArgs a, int64_t w_frags, int64_t x_frags) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  float x[8];
  if (f < w_frags) {
    const float s = pr::exp2i(pr::scale_exp(*a.w_max));
    const int64_t col = column_of(f / a.steps_d * 32 + r, a.F);
    const int step = (int)(f % a.steps_d);
    const int64_t d0 = step * 16 + 8 * h;
    const float* p = a.W + col * a.D + d0;
    if (col >= 0 && d0 + 8 <= a.D) {
      const f32x4 u = *reinterpret_cast<const f32x4u*>(p), w = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = u[e] * s;
        x[4 + e] = w[e] * s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = col >= 0 && d0 + e < a.D ? p[e] * s : 0.f;
    }
    pr::put_frag(a.wp, f / a.steps_d, a.steps_d, step, x);
    return;
  }
  f -= w_frags;
  if (f >= x_frags) return;
  // neighbouring waves take neighbouring row blocks: their reads run along a column
  const int64_t blocks = (a.R + 31) / 32, n = f % blocks * 32 + r;
  const int step = (int)(f / blocks);
  const float s = pr::exp2i(pr::scale_exp(a.scales->x));
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t d = step * 16 + 8 * h + e;
    x[e] = n < a.R && d < a.D ? a.X[a.row0 + n + a.N * d] * s : 0.f;
  }
  pr::put_frag(a.xp, f % blocks, a.steps_d, step, x);
}

// The piece's dZ packed, a wave for a step of 16 hidden features and eight blocks of
// 32 rows; with its column sums where they are wanted.
__global__ void __launch_bounds__(256) ffn_grad_kernel(FfnArgs a) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t groups = (a.R + 255) / 256, blocks = (a.R + 31) / 32;
  const int64_t grp = w % groups;
  const int step = (int)(w / groups);
  if (step >= a.steps_f) return;
  const int64_t f0 = (int64_t)step * 16 + 8 * h;
  const float s = pr::exp2i(pr::scale_exp(a.scales->z));
  float sg[8] = {}, su[8] = {};
  for (int64_t b = grp * 8; b < (grp * 8 + 8 < blocks ? grp * 8 + 8 : blocks); ++b) {
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
}

// db (+)= the sums of the groups of rows, in order
__global__ void __launch_bounds__(256) ffn_db_kernel(FfnArgs a, float* db, int accumulate) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= 2 * a.F) return;
  float s = 0.f;
#pragma unroll 8
  for (int64_t q = 0; q < (a.R + 255) / 256; ++q) s += a.db_part[q * 2 * a.F + v];
  db[v] = accumulate ? db[v] + s : s;
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
  return -pr::scale_exp(a.scales->z) - pr::scale_exp(COLS ? a.scales->x : *a.w_max);
}

// dX (A: W across its rows, B: dZ), COLS false, and dW (A: dZ, B: X, both across
// their rows), COLS true.
template <bool TA, bool TB, bool COLS>
__global__ void __launch_bounds__(pr::GNT, 2) ffn_grads_kernel(pr::GemmArgs g, FfnArgs a, FfnOut o) {
  __shared__ __align__(16) char lds[pr::kGemmLds];
  int tm, tn;
  pr::tile_of((int)blockIdx.x, (g.M + pr::TM - 1) / pr::TM, (g.N + pr::TN - 1) / pr::TN, tm, tn);
  const int t0 = (int)blockIdx.y * g.steps_per_split, t1 = min(g.steps, t0 + g.steps_per_split);
  pr::Acc acc;
  pr::gemm_tile<TA, TB>(g, tm, tn, t0, t1, lds, acc);
  if (o.part) {
    pr::put_tile<false>(acc, tm, tn, g.M, g.N, o.part + (int64_t)blockIdx.y * g.M * g.N, g.N, [](float x) { return x; });
    return;
  }
  const int eo = scale_out<COLS>(a);
  auto value = [&](float x) { return pr::times_exp2(x, eo); };
  if constexpr (!COLS) {
    pr::put_tile<false>(acc, tm, tn, g.M, g.N, o.p, o.ld, value);
  } else {
    // blocks of 32 packed columns lie together in the output: the even ones from its
    // start on, the odd ones from column F on
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = tn * pr::TN + (wave & 3) * 64 + 32 * j + (lane & 31);
      if (n >= g.N) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t blk = (int64_t)tm * (pr::TM / 32) + (wave >> 2) * 4 + i;
        const int64_t f = (blk >> 1) * 32 + 4 * (lane >> 5), left = a.F - f;
        float* q = o.p + n + o.ld * (f + (blk & 1) * a.F);
        auto row = [](int e) { return 8 * (e / 4) + e % 4; };
        if (!o.accumulate) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (row(e) < left) q[o.ld * row(e)] = value(acc.x[i][j][e]);
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

template <bool COLS>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(FfnArgs a, FfnOut o, int M, int N, int splits) {
  const int64_t total = (int64_t)M * N;
  const int eo = scale_out<COLS>(a);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / N, to = COLS ? column_of(m, a.F) : m;
    if (to < 0) continue;
    float x = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) x += o.part[s * total + i];
    float* p = o.p + i % N + o.ld * to;
    x = pr::times_exp2(x, eo);
    *p = o.accumulate ? *p + x : x;
  }
}

int64_t tiles_of(int64_t M, int64_t N) { return (M + pr::TM - 1) / pr::TM * ((N + pr::TN - 1) / pr::TN); }
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
  CNHIP_REQUIRE(N < ((int64_t)1 << 30) && D < ((int64_t)1 << 22) && F < ((int64_t)1 << 28), "%s: too large", who);
  return CNHIP_OK;
}

int run_forward(FfnArgs& a, hipStream_t st, const char* who) {
  const int64_t N = a.N, D = a.D, F = a.F, Fp = pad32(F);
  if (N <= kFewRows) {
    const dim3 grid((unsigned)((F + 7) / 8)), threads(512);
    if (N <= 16) hipLaunchKernelGGL(ffn_few_kernel<1>, grid, threads, 0, st, a);
    else if (N <= 32) hipLaunchKernelGGL(ffn_few_kernel<2>, grid, threads, 0, st, a);
    else hipLaunchKernelGGL(ffn_few_kernel<4>, grid, threads, 0, st, a);
    return check_launch(who);
  }
  a.steps_d = (int)(pad32(D) / 16);
  CNHIP_REQUIRE(tiles_of(2 * Fp, N) < ((int64_t)1 << 31), "%s: too large", who);
  Places w;
  const size_t o_x = w.place((size_t)(pad32(N) * pad32(D)) * 4), o_w = w.place((size_t)(2 * Fp * pad32(D)) * 4),
               o_xe = w.place((size_t)N * 4), o_we = w.place((size_t)(2 * Fp / 32) * 4);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, w.at, &ws, who));
  char* base = static_cast<char*>(ws);
  a.xp = base + o_x;
  a.wp = base + o_w;
  a.xe = reinterpret_cast<int*>(base + o_xe);
  a.we = reinterpret_cast<int*>(base + o_we);
  hipLaunchKernelGGL(ffn_pack_own_kernel, dim3((unsigned)(2 * Fp / 32 + pad32(N) / 32)), dim3(512), 0, st, a,
                     (int)(2 * Fp / 32));
  CNHIP_TRY(check_launch(who));
  const pr::GemmArgs g{pr::Packed{a.wp, (int)(2 * Fp / 32), a.steps_d}, pr::Packed{a.xp, (int)(pad32(N) / 32), a.steps_d},
                       (int)(2 * Fp), (int)N, a.steps_d, a.steps_d, a.steps_d / 2};
  hipLaunchKernelGGL(ffn_forward_kernel, dim3((unsigned)tiles_of(2 * Fp, N)), dim3(pr::GNT), 0, st, g, a);
  return check_launch(who);
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
  const int64_t Rp = pad32(R), pieces = (N + R - 1) / R;
  const pr::Split sx = pr::split_of(D, R, 2 * a.steps_f), sw = pr::split_of(2 * Fp, D, (int)(Rp / 16));
  const size_t px = sx.splits > 1 ? (size_t)sx.splits * (size_t)(D * R) * 4 : 0,
               pw = sw.splits > 1 ? (size_t)sw.splits * (size_t)(2 * Fp * D) * 4 : 0;
  Places w;
  const size_t words = 256 + (size_t)pieces * sizeof(FfnScales);
  const size_t o_max = w.place(words), o_x = w.place((size_t)(Rp * Dp) * 4), o_w = w.place((size_t)(2 * Fp * Dp) * 4),
               o_z = w.place((size_t)(Rp * 2 * Fp) * 4),
               o_db = w.place(db ? (size_t)((R + 255) / 256 * 2 * F) * 4 : 0), o_part = w.place(px > pw ? px : pw);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, w.at, &ws, who));
  char* base = static_cast<char*>(ws);
  a.w_max = reinterpret_cast<uint32_t*>(base + o_max);
  FfnScales* scales = reinterpret_cast<FfnScales*>(base + o_max + 256);
  a.xp = base + o_x;
  a.wp = base + o_w;
  a.zp = base + o_z;
  a.db_part = db ? reinterpret_cast<float*>(base + o_db) : nullptr;
  float* part = reinterpret_cast<float*>(base + o_part);
  CNHIP_TRY(fill_bytes(a.w_max, 0, words, st, who));
  const pr::Packed pw_{a.wp, (int)(2 * Fp / 32), a.steps_d};
  for (int64_t r0 = 0, piece = 0; r0 < N; r0 += R, ++piece) {
    a.row0 = r0;
    a.R = N - r0 < R ? N - r0 : R;
    a.scales = scales + piece;
    const int rb = (int)((a.R + 31) / 32);
    auto clip = [](int64_t n, int64_t most_blocks) { return (int)(n < 1 ? 1 : n > most_blocks ? most_blocks : n); };
    const int64_t chunks = (a.R + 1023) / 1024;
    const int wb = piece ? 0 : clip(2 * D * F / 16384, 512), xb = clip(D * chunks / 4, 512), zb = clip(F * chunks / 2, 2048);
    hipLaunchKernelGGL(ffn_max_kernel, dim3((unsigned)(wb + xb + zb)), dim3(256), 0, st, a, wb, xb);
    CNHIP_TRY(check_launch(who));
    const int64_t wf = piece ? 0 : 2 * Fp / 32 * a.steps_d, xf = (int64_t)rb * a.steps_d;
    hipLaunchKernelGGL(ffn_pack_kernel, dim3((unsigned)((wf + xf + 3) / 4)), dim3(256), 0, st, a, wf, xf);
    CNHIP_TRY(check_launch(who));
    hipLaunchKernelGGL(ffn_grad_kernel, dim3((unsigned)(((a.R + 255) / 256 * a.steps_f + 3) / 4)), dim3(256), 0, st, a);
    CNHIP_TRY(check_launch(who));
    const int add = accumulate || piece > 0;
    if (db) {
      hipLaunchKernelGGL(ffn_db_kernel, dim3((unsigned)((2 * F + 255) / 256)), dim3(256), 0, st, a, db, add);
      CNHIP_TRY(check_launch(who));
    }
    const pr::Packed px_{a.xp, rb, a.steps_d}, pz_{a.zp, rb, 2 * a.steps_f};
    auto product = [&](auto kernel, auto reduce, const pr::Packed& A, const pr::Packed& B, int64_t M, int64_t Nn, int steps,
                       pr::Split sp, FfnOut o) -> int {
      const pr::GemmArgs g{A, B, (int)M, (int)Nn, steps, sp.steps, steps / 2};
      const int splits = (steps + sp.steps - 1) / sp.steps;
      o.part = splits > 1 ? part : nullptr;
      hipLaunchKernelGGL(kernel, dim3((unsigned)tiles_of(M, Nn), (unsigned)splits), dim3(pr::GNT), 0, st, g, a, o);
      CNHIP_TRY(check_launch(who));
      if (splits == 1) return CNHIP_OK;
      hipLaunchKernelGGL(reduce, dim3(elementwise_grid(M * Nn, 256)), dim3(256), 0, st, a, o, (int)M, (int)Nn, splits);
      return check_launch(who);
    };
    CNHIP_TRY(product(ffn_grads_kernel<true, false, false>, ffn_reduce_kernel<false>, pw_, pz_, D, a.R, 2 * a.steps_f, sx,
                      FfnOut{dX + r0, N, nullptr, 0}));
    CNHIP_TRY(product(ffn_grads_kernel<true, true, true>, ffn_reduce_kernel<true>, pz_, px_, 2 * Fp, D, 2 * rb, sw,
                      FfnOut{dW, D, nullptr, add}));
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
  return cnhip::run_backward(a, dX, dW, db, accumulate, cnhip::as_stream(stream), who);
}

}  // extern "C"
