// A Linear to many classes with softmax cross-entropy against class ids, in
// one call that keeps no logits.
//
//   z = X W + b,  lse_n = log sum_v exp(z_nv),
//   loss = sum over the rows with a target of (lse_n - z_n,t) [/ their number],
//   G = (softmax(z) - onehot(t)) [/ their number] for those rows, 0 for others,
//   dX = G W^T,  dW (+)= X^T G,  db (+)= column sums of G.
//
// The rows go through in pieces whose logits fill a bounded workspace: a
// piece's logits are formed, turned into its part of G, and multiplied into dX
// and dW while they are at hand.  Keeping the piece's logits for that moment
// makes three products of 2 N D V flops; forming them again vocabulary piece
// by vocabulary piece would make four.
//
// The products run on the fp16 matrix cores over operands packed as pairs
// (mfma_pair.hpp).  X, W and a piece's G are packed once each and serve two
// products apiece, one along their rows and one across.  The first product
// leaves each row's maximum and sum of exponentials over the 128 columns that
// a wave holds, so the logits are read once more only, to become G.
//
// Bound by the fp16 matrix cores at the clock that the power limit leaves: a large
// library fp16 product reaches 1023 TFLOP/s, a third of which is 341 of fp32
// products.  8192 rows, 1024 -> 32000: logits 1.56 ms (344 TFLOP/s), dX 1.40 ms
// (383), dW 1.56 ms (344), G formed and packed 0.42 ms (5.0 TB/s), everything else
// 0.15 ms; on another card 333, 371 and 338 TFLOP/s.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "mfma_pair.hpp"

namespace cnhip {
namespace {

using pr::f32x16;
using pr::f32x4;
using pr::f32x4u;
using pr::u32x4;

constexpr float kLog2e = 1.4426950408889634f;

// What the kernels of a call share, at the head of its workspace.
struct CeState {
  int held;        // rows of the batch with a target
  uint32_t x_max;  // the largest finite |X| of those rows and |W|, as bits
  uint32_t w_max;
};

struct CeArgs {
  const int32_t* t;
  const float *X, *W, *b;
  int64_t N, D, V;
  int64_t row0, R;     // the piece's first row, and its rows
  float* Z;            // the piece's logits [R, V]
  float2* stat;        // [stat_blocks][R]: maximum and sum of exp(z - maximum)
  int64_t stat_blocks;
  float *lse, *row_loss;
  float2* top;         // of the piece's rows: largest logit, log of the sum of exp(z - largest)
  CeState* state;
  uint32_t *row_max, *w_part;  // largest finite |X| of each row, |W| of each block's part
  int w_blocks;
  int *xe, *we;                // without gradients: the exponents of a row of X, of 32 rows of W^T
  float* zt;                   // and the logit of a row's target
  char *xp, *wp, *gp;  // packed X [N x D], W^T [V x D], the piece's G [R x V]
  int steps_d, steps_v;
  float* db_part;      // [ceil(R / 256)][V], or null
  int32_t* oob;
  int mean;
};

__device__ __forceinline__ bool has_target(const CeArgs& a, int64_t n) {
  const int32_t t = a.t[n];
  return t >= 0 && t < a.V;
}
// The exponent that row n of X is packed with: one for all rows with a target,
// whose products with G are summed, and one of its own for a row without.
__device__ __forceinline__ int x_exp(const CeArgs& a, int64_t n) {
  return pr::scale_exp(has_target(a, n) ? a.state->x_max : a.row_max[n]);
}
// G is 2^kGExp times its value before the division by the number of rows
constexpr int kGExp = 15;
__device__ __forceinline__ float grad_factor(const CeArgs& a) {
  const int held = a.state->held;
  return a.mean ? 1.f / (float)(held > 0 ? held : 1) : 1.f;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  return m;
}

// The largest finite |W| of each of the first w_blocks blocks' parts, then of
// each row of X (64 rows a block, the 16 waves share the columns).
__global__ void __launch_bounds__(1024) ce_max_kernel(CeArgs a) {
  __shared__ uint32_t part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t m = 0;
  if ((int)blockIdx.x < a.w_blocks) {
    const int64_t n = a.V * a.D, n4 = n / 4, step = (int64_t)a.w_blocks * 1024;
    int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x;
    for (; i + 3 * step < n4; i += 4 * step) {
      f32x4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const f32x4u*>(a.W + 4 * (i + u * step));
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[u][e]));
    }
    for (; i < n4; i += step) {
      const f32x4 x = *reinterpret_cast<const f32x4u*>(a.W + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max(m, pr::finite_bits(x[e]));
    }
    if (blockIdx.x == 0 && (int64_t)threadIdx.x < n % 4) m = max(m, pr::finite_bits(a.W[4 * n4 + threadIdx.x]));
    m = wave_max(m);
    if (lane == 0) part[0][wave] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 16; ++w) m = max(m, part[0][w]);
      a.w_part[blockIdx.x] = m;
    }
    return;
  }
  const int64_t n = ((int64_t)blockIdx.x - a.w_blocks) * 64 + lane;
  if (n < a.N) {
    int64_t d = wave;
    for (; d + 7 * 16 < a.D; d += 8 * 16) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = a.X[n + a.N * (d + 16 * u)];
#pragma unroll
      for (int u = 0; u < 8; ++u) m = max(m, pr::finite_bits(x[u]));
    }
    for (; d < a.D; d += 16) m = max(m, pr::finite_bits(a.X[n + a.N * d]));
  }
  part[wave][lane] = m;
  __syncthreads();
  if (wave || n >= a.N) return;
  for (int w = 1; w < 16; ++w) m = max(m, part[w][lane]);
  a.row_max[n] = m;
}

// The call's state (one block): the rows of the batch with a target, the
// largest finite |X| of those, the largest |W|; and the targets past the last
// class added to the caller's count.
__global__ void __launch_bounds__(1024) ce_state_kernel(CeArgs a) {
  __shared__ uint32_t total[4];
  if (threadIdx.x < 4) total[threadIdx.x] = 0;
  __syncthreads();
  int n = 0, past = 0;
  uint32_t x = 0, w = 0;
  constexpr int U = 8;  // loads under way at a time
  for (int64_t i0 = threadIdx.x; i0 < a.N; i0 += U * 1024) {
    int32_t t[U];
    uint32_t m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * 1024;
      t[u] = i < a.N ? a.t[i] : -1;
      m[u] = i < a.N ? a.row_max[i] : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool held = t[u] >= 0 && t[u] < a.V;
      n += held;
      past += t[u] >= a.V;
      if (held) x = max(x, m[u]);
    }
  }
  for (int i = threadIdx.x; i < a.w_blocks; i += 1024) w = max(w, a.w_part[i]);
  x = wave_max(x);
  w = wave_max(w);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    n += __shfl_xor(n, o, 64);
    past += __shfl_xor(past, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    atomicAdd(&total[0], (uint32_t)n);
    atomicAdd(&total[1], (uint32_t)past);
    atomicMax(&total[2], x);
    atomicMax(&total[3], w);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    *a.state = CeState{(int)total[0], total[2], total[3]};
    if (a.oob && total[1]) atomicAdd(a.oob, (int)total[1]);
  }
}

__device__ __forceinline__ void put_frag(char* p, int64_t block, int steps, int step, const float (&x)[8]) {
  u32x4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t h, l;
    pr::split2(x[2 * e], x[2 * e + 1], h, l);
    hi[e] = h;
    lo[e] = l;
  }
  char* q = p + (block * steps + step) * (2 * pr::kFrag) + pr::slot(threadIdx.x & 63, step);
  *reinterpret_cast<u32x4*>(q) = hi;
  *reinterpret_cast<u32x4*>(q + pr::kFrag) = lo;
}

// X and W^T packed, a wave per fragment of 32 rows x 16 k.  Of rows without a
// target only finite values enter: whatever they hold, a zero of G times it is
// zero.
__global__ void __launch_bounds__(256) ce_pack_kernel(CeArgs a, int64_t w_frags, int64_t x_frags) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  float x[8];
  if (f < w_frags) {
    const float s = pr::exp2i(pr::scale_exp(a.state->w_max));
    const int64_t v = f / a.steps_d * 32 + r;
    const int step = (int)(f % a.steps_d);
    const int64_t d0 = step * 16 + 8 * h;
    const float* p = a.W + v * a.D + d0;
    if (v < a.V && d0 + 8 <= a.D) {
      const f32x4 u = *reinterpret_cast<const f32x4u*>(p), w = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = u[e] * s;
        x[4 + e] = w[e] * s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = v < a.V && d0 + e < a.D ? p[e] * s : 0.f;
    }
    put_frag(a.wp, f / a.steps_d, a.steps_d, step, x);
    return;
  }
  f -= w_frags;
  if (f >= x_frags) return;
  // neighbouring waves take neighbouring row blocks: their reads run along a column
  const int64_t blocks = (a.N + 31) / 32, n = f % blocks * 32 + r;
  const int step = (int)(f / blocks);
  const bool in = n < a.N, held = in && has_target(a, n);
  const float s = in ? pr::exp2i(x_exp(a, n)) : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t d = step * 16 + 8 * h + e;
    x[e] = in && d < a.D ? a.X[n + a.N * d] : 0.f;
    if (!held) x[e] = x[e] - x[e] == 0.f ? x[e] : 0.f;
    x[e] *= s;
  }
  put_frag(a.xp, f % blocks, a.steps_d, step, x);
}

// Without gradients no sum runs over blocks of W or rows of X, and each is packed
// with an exponent of its own: one launch, a block of eight waves for 32 rows,
// which reads them twice (the second time from the L2).
__global__ void __launch_bounds__(512) ce_pack_own_kernel(CeArgs a, int w_blocks) {
  __shared__ uint32_t part[8][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const bool w = (int)blockIdx.x < w_blocks;
  const int64_t blk = w ? blockIdx.x : (int64_t)blockIdx.x - w_blocks, row = blk * 32 + r;
  const bool in = row < (w ? a.V : a.N), held = w || (in && has_target(a, row));
  auto load = [&](int step, float (&x)[8]) {
    const int64_t d0 = step * 16 + 8 * h;
    if (w) {
      const float* p = a.W + row * a.D + d0;
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
  if (w) m = wave_max(m);
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
    for (int e = 0; e < 8; ++e) {
      if (!held) x[e] = x[e] - x[e] == 0.f ? x[e] : 0.f;
      x[e] *= f;
    }
    put_frag(w ? a.wp : a.xp, blk, a.steps_d, step, x);
  }
}

// ------------------------------------------------------------- the products
// Element (m, n) of a product goes to out[n + ld m].
struct Out {
  float* p;
  int64_t ld;
  float* part;      // split sums [splits][M][N], or null
  int accumulate;
  int exp_a, exp_b; // which scales to take out: 0 X, 1 W, 2 G
};

__device__ __forceinline__ int scale_of(const CeState& s, int which) {
  return which == 0 ? pr::scale_exp(s.x_max) : which == 1 ? pr::scale_exp(s.w_max) : kGExp;
}
// p[n + ld m] = value(element), or += for ADD, for the elements of a tile that
// this lane holds and that exist.  ADD reads all of a column before it writes
// one, so the reads are under way together.
template <bool ADD, class F>
__device__ __forceinline__ void put_tile(const pr::Acc& acc, int tm, int tn, int M, int N, float* __restrict__ p,
                                         int64_t ld, F&& value) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = tm * pr::TM + (wave >> 2) * 128, m1 = m0 + 4 * (lane >> 5);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = tn * pr::TN + (wave & 3) * 64 + 32 * j + (lane & 31);
    if (n >= N) continue;
    float* q = p + n + ld * m1;
    auto row = [](int i, int e) { return 32 * i + 8 * (e / 4) + e % 4; };
    if (m0 + 128 <= M) {
      float old[4][16];
      if (ADD) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) old[i][e] = q[ld * row(i, e)];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) q[ld * row(i, e)] = ADD ? old[i][e] + value(acc.x[i][j][e]) : value(acc.x[i][j][e]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (m1 + row(i, e) < M) {
            float* at = q + ld * row(i, e);
            *at = ADD ? *at + value(acc.x[i][j][e]) : value(acc.x[i][j][e]);
          }
    }
  }
}

// Logits of a piece (M: classes, N: rows) with each row's maximum and sum of
// exponentials over the wave's 128 classes; stored for the gradients, else the
// targets' alone.
template <bool GRADS>
__global__ void __launch_bounds__(pr::GNT, 2) ce_logits_kernel(pr::GemmArgs g, CeArgs a) {
  __shared__ __align__(16) char lds[pr::kGemmLds];
  int tm, tn;
  pr::tile_of((int)blockIdx.x, (g.M + pr::TM - 1) / pr::TM, (g.N + pr::TN - 1) / pr::TN, tm, tn);
  pr::Acc acc;
  pr::gemm_tile<false, false>(g, tm, tn, 0, g.steps, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = tm * pr::TM + (wave >> 2) * 128;
  if (m0 >= g.M) return;
  int ex[2], ew[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = a.row0 + min(tn * pr::TN + (wave & 3) * 64 + 32 * j + (lane & 31), g.N - 1);
    ex[j] = GRADS ? x_exp(a, n) : a.xe[n];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) ew[i] = GRADS ? pr::scale_exp(a.state->w_max) : a.we[min(m0 / 32 + i, (g.M - 1) / 32)];
  const bool whole = m0 + 128 <= g.M;
  auto row = [&](int i, int e) { return m0 + 32 * i + 8 * (e / 4) + 4 * (lane >> 5) + e % 4; };
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float b = a.b ? a.b[min(row(i, e), g.M - 1)] : 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) acc.x[i][j][e] = pr::times_exp2(acc.x[i][j][e], -ex[j] - ew[i]) + b;
    }
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc.x[i][j][e] = row(i, e) < g.M ? acc.x[i][j][e] : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = tn * pr::TN + (wave & 3) * 64 + 32 * j + (lane & 31);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, acc.x[i][j][e]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sum += __builtin_amdgcn_exp2f((acc.x[i][j][e] - base) * kLog2e);
    sum += __shfl_xor(sum, 32, 64);
    if (n >= g.N) continue;
    if (lane < 32) a.stat[(int64_t)(tm * 2 + (wave >> 2)) * a.R + n] = float2{top, sum};
    if (!GRADS) {
      const int32_t t = a.t[a.row0 + n];
      if (t < m0 || t >= min(m0 + 128, g.M)) continue;
      const int at = t - row(0, 0);  // this lane has it where it is one of row(i, e) - row(0, 0)
      float z = 0.f;
      bool mine = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (at == 32 * i + 8 * (e / 4) + e % 4) {
            z = acc.x[i][j][e];
            mine = true;
          }
      if (mine) a.zt[a.row0 + n] = z;
    }
  }
  if (GRADS) put_tile<false>(acc, tm, tn, g.M, g.N, a.Z, a.R, [](float x) { return x; });
}

// dX (A: W across its rows, B: G) and dW (A: G, B: X, both across their rows)
template <bool TA, bool TB>
__global__ void __launch_bounds__(pr::GNT, 2) ce_grads_kernel(pr::GemmArgs g, CeArgs a, Out o) {
  __shared__ __align__(16) char lds[pr::kGemmLds];
  int tm, tn;
  pr::tile_of((int)blockIdx.x, (g.M + pr::TM - 1) / pr::TM, (g.N + pr::TN - 1) / pr::TN, tm, tn);
  const int t0 = (int)blockIdx.y * g.steps_per_split, t1 = min(g.steps, t0 + g.steps_per_split);
  pr::Acc acc;
  pr::gemm_tile<TA, TB>(g, tm, tn, t0, t1, lds, acc);
  if (o.part) {
    put_tile<false>(acc, tm, tn, g.M, g.N, o.part + (int64_t)blockIdx.y * g.M * g.N, g.N, [](float x) { return x; });
    return;
  }
  const int eo = -scale_of(*a.state, o.exp_a) - scale_of(*a.state, o.exp_b);
  const float factor = grad_factor(a);
  auto value = [&](float x) { return pr::times_exp2(x, eo) * factor; };
  if (o.accumulate) put_tile<true>(acc, tm, tn, g.M, g.N, o.p, o.ld, value);
  else put_tile<false>(acc, tm, tn, g.M, g.N, o.p, o.ld, value);
}

__global__ void __launch_bounds__(256) ce_reduce_kernel(CeArgs a, Out o, int M, int N, int splits) {
  const int64_t total = (int64_t)M * N;
  const int eo = -scale_of(*a.state, o.exp_a) - scale_of(*a.state, o.exp_b);
  const float factor = grad_factor(a);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float x = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) x += o.part[s * total + i];
    float* p = o.p + i % N + o.ld * (i / N);
    x = pr::times_exp2(x, eo) * factor;
    *p = o.accumulate ? *p + x : x;
  }
}

// ------------------------------------------------------------- row by row
// One row's statistics joined: this lane's parts q0, q0 + 16, ... of stat.
__device__ __forceinline__ float2 join_stats(const CeArgs& a, int64_t q0, int64_t rows, int64_t r) {
  float m = -INFINITY, s = 0.f;
  constexpr int U = 8;  // loads under way
  for (; q0 < a.stat_blocks; q0 += 16 * U) {
    float2 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = q0 + 16 * u < a.stat_blocks ? a.stat[(q0 + 16 * u) * rows + r] : float2{-INFINITY, 0.f};
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, x[u].x);
    const float base = top == -INFINITY ? 0.f : top;
    s *= expf(m - base);
#pragma unroll
    for (int u = 0; u < U; ++u) s += x[u].y * expf(x[u].x - base);
    m = top;
  }
  return float2{m, s};
}
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), base = m == -INFINITY ? 0.f : m;
  return float2{m, a.y * expf(a.x - base) + b.y * expf(b.x - base)};
}

// lse and loss of 64 rows a block; the 16 waves share the row's parts.
__global__ void __launch_bounds__(1024) ce_row_kernel(CeArgs a, int grads) {
  __shared__ float2 part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * 64 + lane;
  float2 x = {-INFINITY, 0.f};
  if (r < a.R) x = join_stats(a, wave, a.R, r);
  part[wave][lane] = x;
  __syncthreads();
  if (wave || r >= a.R) return;
  for (int w = 1; w < 16; ++w) x = join(x, part[w][lane]);
  const float log_sum = logf(x.y);
  const int64_t n = a.row0 + r;
  const bool held = has_target(a, n);
  a.lse[n] = x.x + log_sum;
  if (grads) a.top[r] = float2{x.x, log_sum};
  a.row_loss[n] = held ? (x.x - (grads ? a.Z[r + a.R * (int64_t)a.t[n]] : a.zt[n])) + log_sum : 0.f;
}

// The piece's G packed, a wave for a step of 16 classes and eight blocks of 32
// rows; with its column sums where they are wanted.  The softmax is taken from the
// row's largest logit and log sum apart: their sum, the lse, is rounded to 2^-24 of
// itself, which logits of 10^5 and more would feel.
__global__ void __launch_bounds__(256) ce_grad_kernel(CeArgs a) {
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t groups = (a.R + 255) / 256, blocks = (a.R + 31) / 32;
  const int64_t grp = w % groups;
  const int step = (int)(w / groups);
  if (step >= a.steps_v) return;
  const int64_t v0 = (int64_t)step * 16 + 8 * h;
  const float one = pr::exp2i(kGExp);
  float sum[8] = {};
  for (int64_t b = grp * 8; b < (grp * 8 + 8 < blocks ? grp * 8 + 8 : blocks); ++b) {
    const int64_t n = b * 32 + r;
    const bool in = n < a.R;
    const int32_t t = in ? a.t[a.row0 + n] : -1;
    const bool held = t >= 0 && t < a.V;
    const float2 top = in ? a.top[n] : float2{0.f, 0.f};
    const float log2_sum = top.y * kLog2e;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = in && v0 + e < a.V ? a.Z[n + a.R * (v0 + e)] : -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(fmaf(x[e] - top.x, kLog2e, -log2_sum)) - (v0 + e == t ? 1.f : 0.f);
      x[e] = held && v0 + e < a.V ? x[e] * one : 0.f;
      sum[e] += x[e];
    }
    put_frag(a.gp, b, a.steps_v, step, x);
  }
  if (!a.db_part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[e] += __shfl_xor(sum[e], o, 64);
    if (r == 0 && v0 + e < a.V) a.db_part[grp * a.V + v0 + e] = sum[e];
  }
}

// db (+)= the sums of the groups of rows, in order
__global__ void __launch_bounds__(256) ce_db_kernel(CeArgs a, float* db, int accumulate) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= a.V) return;
  float s = 0.f;
  for (int64_t q = 0; q < (a.R + 255) / 256; ++q) s += a.db_part[q * a.V + v];
  s = pr::times_exp2(s, -kGExp) * grad_factor(a);
  db[v] = accumulate ? db[v] + s : s;
}

// The losses of the rows in a fixed order (one block); `count`: also the targets
// past the last class, where no state kernel does.
__global__ void __launch_bounds__(1024) ce_loss_kernel(CeArgs a, float* __restrict__ loss, int count) {
  __shared__ float part[16];
  __shared__ int total[2];
  if (threadIdx.x < 2) total[threadIdx.x] = 0;
  __syncthreads();
  float s = 0.f;
  int n = 0, past = 0;
  constexpr int U = 8;  // loads under way
  for (int64_t i0 = threadIdx.x; i0 < a.N; i0 += U * 1024) {
    float l[U];
    int32_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * 1024;
      l[u] = i < a.N ? a.row_loss[i] : 0.f;
      t[u] = i < a.N ? a.t[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s += l[u];
      n += t[u] >= 0 && t[u] < a.V;
      past += t[u] >= a.V;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
    past += __shfl_xor(past, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    part[threadIdx.x >> 6] = s;
    atomicAdd(&total[0], n);
    atomicAdd(&total[1], past);
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) s += part[w];
  *loss = a.mean ? s / (float)(total[0] > 0 ? total[0] : 1) : s;
  if (count && a.oob && total[1]) atomicAdd(a.oob, total[1]);
}

// ------------------------------------------------------------ few rows
// Up to kFewRows rows are one or two columns of 32 lanes: W is then read once or
// twice and each value used for a handful of products, so the fp32 matrix cores
// keep up with memory and nothing is packed.  Four launches: logits with row
// statistics, the rows' losses, G with dW, db and parts of dX, and the sum of
// those parts.  64 rows, 512 -> 8192 with gradients: 49 us (15, 7, 26 and 5), of
// which the fp32 products alone take 10 and the memory 7; 64 against 65 rows, this
// way and packed: forward 21 and 55 us, with gradients 52 and 110; 1024 -> 32000 95
// and 140, 277 and 256, where the parts of dX are as many bytes as W.
constexpr int kFewRows = 64;
constexpr int kFewClasses = 32;   // classes a block of the first launch
constexpr int kFewSlice = 64;     // classes a block of the third
constexpr int kFewWidth = 128;    // features a block of the third: 32 a wave

// 32 classes; the eight waves share out the features, a step of 16 each.
template <int NB>
__global__ void __launch_bounds__(512) ce_few_logits_kernel(CeArgs a) {
  __shared__ float part[8][kFewClasses][64 + 1];
  __shared__ float2 stat[8][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, r = lane & 31;
  const int64_t v0 = (int64_t)blockIdx.x * kFewClasses, v = v0 + r;
  const int N = (int)a.N, steps = (int)((a.D + 15) / 16);
  bool held[NB], in[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    in[j] = 32 * j + r < N;
    held[j] = in[j] && has_target(a, 32 * j + r);
  }
  float w[2][8], x[2][NB][8];
  auto load = [&](int s, int b) {
    const int64_t d0 = 16 * (int64_t)s + 8 * h;
    const float* p = a.W + v * a.D + d0;
    if (v < a.V && d0 + 8 <= a.D) {
      const f32x4 lo = *reinterpret_cast<const f32x4u*>(p), hi = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[b][e] = lo[e];
        w[b][4 + e] = hi[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[b][e] = v < a.V && d0 + e < a.D ? p[e] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[b][j][e] = in[j] && d0 + e < a.D ? a.X[32 * j + r + a.N * (d0 + e)] : 0.f;
  };
  f32x16 acc[NB] = {};
  auto multiply = [&](int b) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float y = x[b][j][e];
        if (!held[j]) y = y - y == 0.f ? y : 0.f;
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(w[b][e], y, acc[j], 0, 0, 0);
      }
  };
  if (wave < steps) load(wave, 0);
  for (int s = wave; s < steps; s += 16) {
    if (s + 8 < steps) load(s + 8, 1);
    multiply(0);
    if (s + 16 < steps) load(s + 16, 0);
    if (s + 8 < steps) multiply(1);
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) part[wave][8 * (e / 4) + 4 * h + e % 4][32 * j + r] = acc[j][e];
  __syncthreads();
  // a lane per row, four classes a wave
  const int n = lane;
  float z[4], top = -INFINITY;
  if (n < 32 * NB) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 4 * wave + e;
      z[e] = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) z[e] += part[q][c][n];
      if (a.b && v0 + c < a.V) z[e] += a.b[v0 + c];
      if (v0 + c >= a.V) z[e] = -INFINITY;
      else if (n < N) a.Z[n + a.N * (v0 + c)] = z[e];
      top = fmaxf(top, z[e]);
    }
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += expf(z[e] - base);
    stat[wave][n] = float2{top, sum};
  }
  __syncthreads();
  if (wave || n >= N) return;
  float m = -INFINITY, t = 0.f;
  for (int q = 0; q < 8; ++q) m = fmaxf(m, stat[q][n].x);
  const float base = m == -INFINITY ? 0.f : m;
  for (int q = 0; q < 8; ++q) t += stat[q][n].y * expf(stat[q][n].x - base);
  a.stat[(int64_t)blockIdx.x * a.N + n] = float2{m, t};
}

// The rows' log-sum-exp and losses, their number and sum (one block).
__global__ void __launch_bounds__(1024) ce_few_rows_kernel(CeArgs a, float* __restrict__ loss) {
  __shared__ float2 part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float2 x = {-INFINITY, 0.f};
  if (lane < a.N) x = join_stats(a, wave, a.N, lane);
  part[wave][lane] = x;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < 16; ++w) x = join(x, part[w][lane]);
  const int32_t t = lane < a.N ? a.t[lane] : -1;
  const bool held = t >= 0 && t < a.V;
  const float log_sum = logf(x.y);
  if (lane < a.N) {
    a.lse[lane] = x.x + log_sum;
    a.top[lane] = float2{x.x, log_sum};
  }
  float l = held ? (x.x - a.Z[lane + a.N * (int64_t)t]) + log_sum : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  const int count = __popcll(__ballot(held)), past = __popcll(__ballot(t >= a.V));
  if (lane == 0) {
    a.state->held = count;
    *loss = a.mean ? l / (float)(count > 0 ? count : 1) : l;
    if (a.oob && past) atomicAdd(a.oob, past);
  }
}

// A slice of classes and 128 features, 32 a wave: G of the slice in LDS, dW and
// db of it, and its part of dX ([slice][feature][row]).
template <int NB>
__global__ void __launch_bounds__(256) ce_few_grads_kernel(CeArgs a, float* dW, float* db, float* part, int accumulate) {
  constexpr int NR = 32 * NB, LD = NR + 1;
  __shared__ float G[kFewSlice * LD], xs[kFewWidth * LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, r = lane & 31;
  const int64_t v0 = (int64_t)blockIdx.x * kFewSlice, d0 = (int64_t)blockIdx.y * kFewWidth, d = d0 + 32 * wave + r;
  const int N = (int)a.N;
  const float f = grad_factor(a);
  // W of the wave's features, and everything else that is read, goes out first
  float w[kFewSlice / 2];
#pragma unroll
  for (int s = 0; s < kFewSlice / 2; ++s) {
    const int64_t v = v0 + 2 * s + h;
    w[s] = d < a.D && v < a.V ? a.W[d + a.D * v] : 0.f;
  }
  {
    const int n = threadIdx.x % NR;
    const int32_t t = n < N ? a.t[n] : -1;
    const bool held = t >= 0 && t < a.V;
    const float2 top = held ? a.top[n] : float2{0.f, 0.f};
    constexpr int STEP = 256 / NR, UG = kFewSlice / STEP, UX = kFewWidth / STEP;
    float z[UG], x[UX];
#pragma unroll
    for (int u = 0; u < UG; ++u) {
      const int64_t v = v0 + threadIdx.x / NR + u * STEP;
      z[u] = held && v < a.V ? a.Z[n + a.N * v] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < UX; ++u) {
      const int64_t dx = d0 + threadIdx.x / NR + u * STEP;
      x[u] = held && dx < a.D ? a.X[n + a.N * dx] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < UG; ++u) {
      const int c = threadIdx.x / NR + u * STEP;
      const int64_t v = v0 + c;
      G[c * LD + n] = held && v < a.V ? (expf((z[u] - top.x) - top.y) - (v == t ? 1.f : 0.f)) * f : 0.f;
    }
#pragma unroll
    for (int u = 0; u < UX; ++u) xs[(threadIdx.x / NR + u * STEP) * LD + n] = x[u];
  }
  __syncthreads();
  // dX's part: W's features over the classes
  f32x16 acc[NB] = {};
#pragma unroll
  for (int s = 0; s < kFewSlice / 2; ++s)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(w[s], G[(2 * s + h) * LD + 32 * j + r], acc[j], 0, 0, 0);
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t m = d0 + 32 * wave + 8 * (e / 4) + 4 * h + e % 4;
      if (m < a.D && 32 * j + r < N) part[((int64_t)blockIdx.x * a.D + m) * a.N + 32 * j + r] = acc[j][e];
    }
  // dW: G over the rows of the batch
  constexpr int C = kFewSlice / 32;
  f32x16 dw[C] = {};
#pragma unroll 16
  for (int s = 0; s < NR / 2; ++s) {
    const float x = xs[(32 * wave + r) * LD + 2 * s + h];
#pragma unroll
    for (int i = 0; i < C; ++i)
      dw[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(G[(32 * i + r) * LD + 2 * s + h], x, dw[i], 0, 0, 0);
  }
  if (d < a.D) {
    float* p = dW + d + a.D * (v0 + 4 * h);
    const int64_t left = a.V - (v0 + 4 * h);
    auto row = [](int i, int e) { return 32 * i + 8 * (e / 4) + e % 4; };
    float old[C][16];
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) old[i][e] = accumulate && row(i, e) < left ? p[a.D * row(i, e)] : 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (row(i, e) < left) p[a.D * row(i, e)] = old[i][e] + dw[i][e];
  }
  if (db && blockIdx.y == 0 && threadIdx.x < kFewSlice && v0 + threadIdx.x < a.V) {
    float sum = 0.f;
    for (int n = 0; n < NR; ++n) sum += G[threadIdx.x * LD + n];
    float* p = db + v0 + threadIdx.x;
    *p = accumulate ? *p + sum : sum;
  }
}

// dX = the slices' parts, in order
__global__ void __launch_bounds__(256) ce_few_dx_kernel(const float* __restrict__ part, float* __restrict__ dX, int64_t n,
                                                        int slices) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 16
  for (int q = 0; q < slices; ++q) s += part[q * n + i];
  dX[i] = s;
}

struct CeGrads {
  float *dX, *dW, *db;
  int accumulate;
};

struct Split {
  int splits, steps;
};
// Splits of a contraction so that the tiles fill the 256 CUs, each at least 16
// steps (256 k) long.
Split split_of(int64_t M, int64_t N, int steps) {
  const int64_t tiles = (M + pr::TM - 1) / pr::TM * ((N + pr::TN - 1) / pr::TN);
  int64_t s = tiles >= 224 ? 1 : 256 / tiles;
  if (s > steps / 16) s = steps / 16;
  if (s < 1) s = 1;
  int per = (int)((steps + s - 1) / s);
  per = (per + 1) / 2 * 2;
  return Split{(steps + per - 1) / per, per};
}

int run_few(CeArgs& a, float* loss, const CeGrads* g, hipStream_t st, const char* who) {
  const int64_t N = a.N, D = a.D, V = a.V, slices = (V + kFewSlice - 1) / kFewSlice;
  a.stat_blocks = (V + kFewClasses - 1) / kFewClasses;
  const size_t z = (size_t)(N * V) * 4, stat = (size_t)(a.stat_blocks * N) * 8, part = g ? (size_t)(slices * D * N) * 4 : 0;
  void* ws = nullptr;
  constexpr size_t head = 256 + kFewRows * sizeof(float2);  // the state, the rows' statistics
  CNHIP_TRY(scratch(st, kScratchLayer, head + stat + z + part, &ws, who));
  a.state = static_cast<CeState*>(ws);
  a.top = reinterpret_cast<float2*>(static_cast<char*>(ws) + 256);
  a.stat = reinterpret_cast<float2*>(static_cast<char*>(ws) + head);
  a.Z = reinterpret_cast<float*>(a.stat + a.stat_blocks * N);
  float* dx_part = a.Z + N * V;
  const dim3 logits((unsigned)a.stat_blocks), grads((unsigned)slices, (unsigned)((D + kFewWidth - 1) / kFewWidth));
  if (N <= 32) hipLaunchKernelGGL(ce_few_logits_kernel<1>, logits, dim3(512), 0, st, a);
  else hipLaunchKernelGGL(ce_few_logits_kernel<2>, logits, dim3(512), 0, st, a);
  CNHIP_TRY(check_launch(who));
  hipLaunchKernelGGL(ce_few_rows_kernel, dim3(1), dim3(1024), 0, st, a, loss);
  CNHIP_TRY(check_launch(who));
  if (!g) return CNHIP_OK;
  if (N <= 32) hipLaunchKernelGGL(ce_few_grads_kernel<1>, grads, dim3(256), 0, st, a, g->dW, g->db, dx_part, g->accumulate);
  else hipLaunchKernelGGL(ce_few_grads_kernel<2>, grads, dim3(256), 0, st, a, g->dW, g->db, dx_part, g->accumulate);
  CNHIP_TRY(check_launch(who));
  hipLaunchKernelGGL(ce_few_dx_kernel, dim3((unsigned)((N * D + 255) / 256)), dim3(256), 0, st, dx_part, g->dX, N * D,
                     (int)slices);
  return check_launch(who);
}

int run(const float* X, const float* W, const float* b, const int32_t* targets, float* loss, float* lse,
        const CeGrads* g, int64_t N, int64_t D, int64_t V, int reduction, int32_t* oob, hipStream_t st,
        const char* who) {
  CNHIP_REQUIRE(N > 0 && D > 0 && V > 0, "%s: bad shape batch=%lld in_features=%lld classes=%lld", who, (long long)N,
                (long long)D, (long long)V);
  CNHIP_REQUIRE(X && W && targets && loss && lse, "%s: NULL pointer", who);
  CNHIP_REQUIRE(reduction == CNHIP_REDUCE_MEAN || reduction == CNHIP_REDUCE_SUM, "%s: bad reduction %d", who, reduction);
  CNHIP_REQUIRE(V < ((int64_t)1 << 30) && N < ((int64_t)1 << 30) && D < ((int64_t)1 << 22), "%s: too large", who);
  if (g) {
    CNHIP_REQUIRE(g->dX && g->dW, "%s: NULL pointer", who);
    CNHIP_REQUIRE(!b == !g->db, "%s: db goes with b", who);
    CNHIP_REQUIRE(g->accumulate == 0 || g->accumulate == 1, "%s: accumulate must be 0 or 1", who);
  }
  CeArgs a{};
  a.t = targets;
  a.X = X;
  a.W = W;
  a.b = b;
  a.N = N;
  a.D = D;
  a.V = V;
  a.lse = lse;
  a.oob = oob;
  a.mean = reduction == CNHIP_REDUCE_MEAN;
  if (N <= kFewRows) return run_few(a, loss, g, st, who);
  a.steps_d = (int)((D + 31) / 32 * 2);
  a.steps_v = (int)((V + 31) / 32 * 2);
  a.stat_blocks = (V + 127) / 128;
  // Rows of a piece: 2^27 logits (half a GiB, and as much for G), but 1024 rows
  // at least, so that the gradients of W are read and written once in 1024 rows
  // at most.  8192 rows, 1024 -> 32000: 2^26 4.98 ms, 2^27 4.61, 2^28 4.46.
  const int64_t most = ((int64_t)1 << 27) / V;
  int64_t R = most < 1024 ? 1024 : most / 256 * 256;
  if (R > N) R = N;
  const int64_t Rp = (R + 31) / 32 * 32, Np = (N + 31) / 32 * 32, Vp = (V + 31) / 32 * 32, Dp = (D + 31) / 32 * 32;
  const Split sx = split_of(D, R, a.steps_v), sw = split_of(V, D, (int)(Rp / 16));
  const int64_t wb = V * D / (16 * 1024);  // 16 values a thread and more
  a.w_blocks = (int)(wb < 1 ? 1 : wb > 1024 ? 1024 : wb);
  size_t at = 0;
  auto place = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t o_state = place(sizeof(CeState)), o_loss = place((size_t)N * 4), o_rows = place((size_t)N * 4),
               o_wpart = place((size_t)a.w_blocks * 4), o_x = place((size_t)(Np * Dp) * 4),
               o_w = place((size_t)(Vp * Dp) * 4), o_z = place(g ? (size_t)R * (size_t)V * 4 : 0),
               o_stat = place((size_t)a.stat_blocks * (size_t)R * 8), o_xe = place(g ? 0 : (size_t)N * 4),
               o_we = place(g ? 0 : (size_t)(Vp / 32) * 4), o_zt = place(g ? 0 : (size_t)N * 4);
  const size_t o_top = place(g ? (size_t)R * sizeof(float2) : 0);
  const size_t o_g = place(g ? (size_t)(Rp * Vp) * 4 : 0), o_db = place(g && g->db ? (size_t)((R + 255) / 256 * V) * 4 : 0);
  const size_t px = sx.splits > 1 ? (size_t)sx.splits * (size_t)(D * R) * 4 : 0,
               pw = sw.splits > 1 ? (size_t)sw.splits * (size_t)(V * D) * 4 : 0;
  const size_t o_part = place(g ? (px > pw ? px : pw) : 0);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, at, &ws, who));
  char* base = static_cast<char*>(ws);
  a.state = reinterpret_cast<CeState*>(base + o_state);
  a.row_loss = reinterpret_cast<float*>(base + o_loss);
  a.row_max = reinterpret_cast<uint32_t*>(base + o_rows);
  a.w_part = reinterpret_cast<uint32_t*>(base + o_wpart);
  a.xp = base + o_x;
  a.wp = base + o_w;
  a.Z = reinterpret_cast<float*>(base + o_z);
  a.stat = reinterpret_cast<float2*>(base + o_stat);
  a.gp = base + o_g;
  a.xe = reinterpret_cast<int*>(base + o_xe);
  a.we = reinterpret_cast<int*>(base + o_we);
  a.zt = reinterpret_cast<float*>(base + o_zt);
  a.top = reinterpret_cast<float2*>(base + o_top);
  a.db_part = g && g->db ? reinterpret_cast<float*>(base + o_db) : nullptr;
  float* part = reinterpret_cast<float*>(base + o_part);

  if (g) {
    hipLaunchKernelGGL(ce_max_kernel, dim3((unsigned)(a.w_blocks + (N + 63) / 64)), dim3(1024), 0, st, a);
    CNHIP_TRY(check_launch(who));
    hipLaunchKernelGGL(ce_state_kernel, dim3(1), dim3(1024), 0, st, a);
    CNHIP_TRY(check_launch(who));
    const int64_t w_frags = Vp / 32 * a.steps_d, x_frags = Np / 32 * a.steps_d;
    hipLaunchKernelGGL(ce_pack_kernel, dim3((unsigned)((w_frags + x_frags + 3) / 4)), dim3(256), 0, st, a, w_frags, x_frags);
    CNHIP_TRY(check_launch(who));
  } else {
    hipLaunchKernelGGL(ce_pack_own_kernel, dim3((unsigned)((Vp + Np) / 32)), dim3(512), 0, st, a, (int)(Vp / 32));
    CNHIP_TRY(check_launch(who));
  }

  const pr::Packed pw_{a.wp, (int)(Vp / 32), a.steps_d};
  auto tiles = [](int64_t M, int64_t Nn) { return (M + pr::TM - 1) / pr::TM * ((Nn + pr::TN - 1) / pr::TN); };
  for (int64_t r0 = 0; r0 < N; r0 += R) {
    a.row0 = r0;
    a.R = N - r0 < R ? N - r0 : R;
    const int rb = (int)((a.R + 31) / 32);
    const pr::Packed px_{a.xp + (r0 / 32) * a.steps_d * (2 * pr::kFrag), rb, a.steps_d};
    const pr::Packed pg_{a.gp, rb, a.steps_v};
    {
      const pr::GemmArgs ga{pw_, px_, (int)V, (int)a.R, a.steps_d, a.steps_d, a.steps_d / 2};
      const dim3 grid((unsigned)tiles(V, a.R));
      if (g) hipLaunchKernelGGL(ce_logits_kernel<true>, grid, dim3(pr::GNT), 0, st, ga, a);
      else hipLaunchKernelGGL(ce_logits_kernel<false>, grid, dim3(pr::GNT), 0, st, ga, a);
      CNHIP_TRY(check_launch(who));
    }
    hipLaunchKernelGGL(ce_row_kernel, dim3((unsigned)((a.R + 63) / 64)), dim3(1024), 0, st, a, g ? 1 : 0);
    CNHIP_TRY(check_launch(who));
    if (!g) continue;
    const int add = g->accumulate || r0 > 0;
    hipLaunchKernelGGL(ce_grad_kernel, dim3((unsigned)(((a.R + 255) / 256 * a.steps_v + 3) / 4)), dim3(256), 0, st, a);
    CNHIP_TRY(check_launch(who));
    if (g->db) {
      hipLaunchKernelGGL(ce_db_kernel, dim3((unsigned)((V + 255) / 256)), dim3(256), 0, st, a, g->db, add);
      CNHIP_TRY(check_launch(who));
    }
    auto grads = [&](auto kernel, const pr::Packed& A, const pr::Packed& B, int64_t M, int64_t Nn, int steps, Split sp,
                     Out o) -> int {
      const pr::GemmArgs ga{A, B, (int)M, (int)Nn, steps, sp.steps, steps / 2};
      const int splits = (steps + sp.steps - 1) / sp.steps;
      o.part = splits > 1 ? part : nullptr;
      hipLaunchKernelGGL(kernel, dim3((unsigned)tiles(M, Nn), (unsigned)splits), dim3(pr::GNT), 0, st, ga, a, o);
      CNHIP_TRY(check_launch(who));
      if (splits == 1) return CNHIP_OK;
      hipLaunchKernelGGL(ce_reduce_kernel, dim3(elementwise_grid(M * Nn, 256)), dim3(256), 0, st, a, o, (int)M, (int)Nn,
                         splits);
      return check_launch(who);
    };
    CNHIP_TRY(grads(ce_grads_kernel<true, false>, pw_, pg_, D, a.R, a.steps_v, sx,
                    Out{g->dX + r0, N, nullptr, 0, 1, 2}));
    CNHIP_TRY(grads(ce_grads_kernel<true, true>, pg_, px_, V, D, 2 * rb, sw, Out{g->dW, D, nullptr, add, 0, 2}));
  }
  hipLaunchKernelGGL(ce_loss_kernel, dim3(1), dim3(1024), 0, st, a, loss, g ? 0 : 1);
  return check_launch(who);
}

}  // namespace
}  // namespace cnhip

extern "C" {

int cnhip_linear_ce_forward(const float* X, const float* W, const float* b, const int32_t* targets, float* loss,
                            float* lse, int64_t batch, int64_t in_features, int64_t classes, int reduction,
                            int32_t* oob_count, cnhip_stream_t stream) {
  return cnhip::run(X, W, b, targets, loss, lse, nullptr, batch, in_features, classes, reduction, oob_count,
                    cnhip::as_stream(stream), "cnhip_linear_ce_forward");
}

int cnhip_linear_ce_head(const float* X, const float* W, const float* b, const int32_t* targets, float* loss,
                         float* lse, float* dX, float* dW, float* db, int64_t batch, int64_t in_features,
                         int64_t classes, int reduction, int accumulate, int32_t* oob_count, cnhip_stream_t stream) {
  const cnhip::CeGrads g{dX, dW, db, accumulate};
  return cnhip::run(X, W, b, targets, loss, lse, &g, batch, in_features, classes, reduction, oob_count,
                    cnhip::as_stream(stream), "cnhip_linear_ce_head");
}

}  // extern "C"
