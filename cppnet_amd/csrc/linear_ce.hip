// A Linear to many classes with softmax cross-entropy against class ids, in
// one call that keeps no logits.
//
//   z = X W + b,  lse_n = log sum_v exp(z_nv),
//   loss = sum over the rows with a target of (lse_n - z_n,t) [/ their number],
//   G = (softmax(z) - onehot(t)) [/ their number] for those rows, 0 for others,
//   dX = G W^T,  dW (+)= X^T G,  db (+)= column sums of G.
//
// The rows go through in pieces whose logits fill a bounded workspace: a
// piece's logits are formed, turned into its part of G where they lie, and
// multiplied into dX and dW while they are at hand.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace cnhip {

int gemm_f32(int trans_a, int trans_b, int64_t M, int64_t N, int64_t K, float alpha, const float* A, int64_t lda,
             const float* B, int64_t ldb, float beta, float* C, int64_t ldc, const float* bias, int epilogue,
             hipStream_t st, const char* who);

namespace {

constexpr int kStatCols = 64;  // columns that a wave reduces for its rows

struct CeArgs {
  const int32_t* t;
  int64_t N, V;
  int64_t row0, R;     // the piece's first row, and its rows
  float* Z;            // the piece's logits [R, V]
  float2* stat;        // [col blocks][R]: maximum and sum of exp(z - maximum)
  int64_t stat_blocks;
  float *lse, *row_loss;
  int* held;           // rows of the batch with a target
  int32_t* oob;
  int mean;
};

// Rows of the batch with a target (one block), and the count of targets past
// the last class.
__global__ void __launch_bounds__(1024) ce_count_kernel(const int32_t* __restrict__ t, int64_t N, int64_t V, int* held,
                                                        int32_t* oob) {
  __shared__ int total[2];
  if (threadIdx.x < 2) total[threadIdx.x] = 0;
  __syncthreads();
  int n = 0, past = 0;
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    n += t[i] >= 0 && t[i] < V;
    past += t[i] >= V;
  }
  atomicAdd(&total[0], n);
  atomicAdd(&total[1], past);
  __syncthreads();
  if (threadIdx.x == 0) {
    *held = total[0];
    if (oob && total[1]) atomicAdd(oob, total[1]);
  }
}

// a lane per row, kStatCols columns
__global__ void __launch_bounds__(64) ce_stat_kernel(CeArgs a) {
  const int64_t r = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (r >= a.R) return;
  const int64_t c0 = (int64_t)blockIdx.y * kStatCols, c1 = c0 + kStatCols < a.V ? c0 + kStatCols : a.V;
  float m = -INFINITY, s = 0.f;
  for (int64_t c = c0; c < c1; ++c) {
    const float z = a.Z[r + a.R * c], mn = fmaxf(m, z), base = mn == -INFINITY ? 0.f : mn;
    s = s * expf(m - base) + expf(z - base);
    m = mn;
  }
  a.stat[(int64_t)blockIdx.y * a.R + r] = float2{m, s};
}

__global__ void __launch_bounds__(64) ce_row_kernel(CeArgs a) {
  const int64_t r = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (r >= a.R) return;
  float m = -INFINITY, s = 0.f;
  for (int64_t q = 0; q < a.stat_blocks; ++q) {
    const float2 x = a.stat[q * a.R + r];
    const float mn = fmaxf(m, x.x), base = mn == -INFINITY ? 0.f : mn;
    s = s * expf(m - base) + x.y * expf(x.x - base);
    m = mn;
  }
  const float lse = m + logf(s);
  const int32_t t = a.t[a.row0 + r];
  a.lse[a.row0 + r] = lse;
  a.row_loss[a.row0 + r] = t >= 0 && t < a.V ? lse - a.Z[r + a.R * (int64_t)t] : 0.f;
}

// Z -> G where it lies
__global__ void __launch_bounds__(256) ce_grad_kernel(CeArgs a) {
  const int64_t total = a.R * a.V;
  const int held = *a.held;
  const float f = a.mean ? 1.f / (float)(held > 0 ? held : 1) : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i % a.R, c = i / a.R;
    const int32_t t = a.t[a.row0 + r];
    float g = 0.f;
    if (t >= 0 && t < a.V) g = (expf(a.Z[i] - a.lse[a.row0 + r]) - (c == t ? 1.f : 0.f)) * f;
    a.Z[i] = g;
  }
}

// the losses of the rows in a fixed order (one block)
__global__ void __launch_bounds__(1024) ce_loss_kernel(const float* __restrict__ row_loss, int64_t N,
                                                       const int* __restrict__ held, int mean,
                                                       float* __restrict__ loss) {
  __shared__ float part[1024];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024) s += row_loss[i];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int w = 512; w > 0; w >>= 1) {
    if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = mean ? part[0] / (float)(*held > 0 ? *held : 1) : part[0];
}

struct CeGrads {
  float *dX, *dW, *db;
  int accumulate;
};

int run(const float* X, const float* W, const float* b, const int32_t* targets, float* loss, float* lse,
        const CeGrads* g, int64_t N, int64_t D, int64_t V, int reduction, int32_t* oob, hipStream_t st,
        const char* who) {
  CNHIP_REQUIRE(N > 0 && D > 0 && V > 0, "%s: bad shape batch=%lld in_features=%lld classes=%lld", who, (long long)N,
                (long long)D, (long long)V);
  CNHIP_REQUIRE(X && W && targets && loss && lse, "%s: NULL pointer", who);
  CNHIP_REQUIRE(reduction == CNHIP_REDUCE_MEAN || reduction == CNHIP_REDUCE_SUM, "%s: bad reduction %d", who, reduction);
  CNHIP_REQUIRE(V < ((int64_t)1 << 31) && N < ((int64_t)1 << 31) && D < ((int64_t)1 << 31), "%s: too large", who);
  if (g) {
    CNHIP_REQUIRE(g->dX && g->dW, "%s: NULL pointer", who);
    CNHIP_REQUIRE(!b == !g->db, "%s: db goes with b", who);
    CNHIP_REQUIRE(g->accumulate == 0 || g->accumulate == 1, "%s: accumulate must be 0 or 1", who);
  }
  CeArgs a{};
  a.t = targets;
  a.N = N;
  a.V = V;
  a.lse = lse;
  a.oob = oob;
  a.mean = reduction == CNHIP_REDUCE_MEAN;
  a.stat_blocks = (V + kStatCols - 1) / kStatCols;
  CNHIP_REQUIRE(a.stat_blocks <= 65535, "%s: too many classes", who);
  const int64_t most = (int64_t)1 << 28;  // logits of a piece
  int64_t R = most / V;
  R = R < 1 ? 1 : R >= N ? N : R >= 256 ? R / 256 * 256 : R;
  const size_t z = (size_t)R * (size_t)V * sizeof(float), s = (size_t)a.stat_blocks * (size_t)R * sizeof(float2);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, z + 16 + s + (size_t)N * sizeof(float) + 16, &ws, who));
  char* p = static_cast<char*>(ws);
  a.Z = reinterpret_cast<float*>(p);
  a.stat = reinterpret_cast<float2*>(p + (z + 15) / 16 * 16);
  a.row_loss = reinterpret_cast<float*>(a.stat + a.stat_blocks * R);
  a.held = reinterpret_cast<int*>(a.row_loss + N);
  hipLaunchKernelGGL(ce_count_kernel, dim3(1), dim3(1024), 0, st, targets, N, V, a.held, oob);
  CNHIP_TRY(check_launch(who));
  for (int64_t r0 = 0; r0 < N; r0 += R) {
    a.row0 = r0;
    a.R = N - r0 < R ? N - r0 : R;
    CNHIP_TRY(gemm_f32(0, 0, a.R, V, D, 1.f, X + r0, N, W, D, 0.f, a.Z, a.R, b, 0, st, who));
    hipLaunchKernelGGL(ce_stat_kernel, dim3((unsigned)((a.R + 63) / 64), (unsigned)a.stat_blocks), dim3(64), 0, st, a);
    CNHIP_TRY(check_launch(who));
    hipLaunchKernelGGL(ce_row_kernel, dim3((unsigned)((a.R + 63) / 64)), dim3(64), 0, st, a);
    CNHIP_TRY(check_launch(who));
    if (!g) continue;
    hipLaunchKernelGGL(ce_grad_kernel, dim3(elementwise_grid(a.R * V, 256)), dim3(256), 0, st, a);
    CNHIP_TRY(check_launch(who));
    const int add = g->accumulate || r0 > 0;
    CNHIP_TRY(gemm_f32(0, 1, a.R, D, V, 1.f, a.Z, a.R, W, D, 0.f, g->dX + r0, N, nullptr, 0, st, who));
    CNHIP_TRY(gemm_f32(1, 0, D, V, a.R, 1.f, X + r0, N, a.Z, a.R, add ? 1.f : 0.f, g->dW, D, nullptr, 0, st, who));
    if (g->db) CNHIP_TRY(cnhip_column_sum(a.Z, g->db, a.R, V, add, st));
  }
  hipLaunchKernelGGL(ce_loss_kernel, dim3(1), dim3(1024), 0, st, a.row_loss, N, a.held, a.mean, loss);
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
