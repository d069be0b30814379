// Token embedding with a scale, and its gradient by sorted tokens.
//
//   out[p, d] = scale * Wt[d + D id_p]
//   gWt[d + D v] (+)= scale * sum over the rows p with id_p = v of dY[p, d]
//
// The table is token-major, which is also the ColMajor [D, V] weight of a
// Linear from D features to V logits: a model with tied weights uses one
// buffer for both, and the accumulating form adds the lookup's gradient to the
// Linear's.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace cnhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t i32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Row of the sequence that the id at j = b + B s belongs to, and the reverse.
__device__ __forceinline__ int64_t row_of(int64_t j, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? j : j / B + S * (j % B);
}
__device__ __forceinline__ int64_t id_of(int64_t p, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? p : p / S + B * (p % S);
}

// A tile of 64 rows x 64 features: read along the features of the table,
// turned in LDS, written along the rows of out.
__global__ void __launch_bounds__(256) token_fwd_kernel(const int32_t* __restrict__ ids, const float* __restrict__ Wt,
                                                        float* __restrict__ out, int64_t B, int64_t S, int64_t V,
                                                        int64_t D, float scale, int rows, int32_t* __restrict__ oob) {
  __shared__ float tile[64][65];
  __shared__ int64_t tok[64];
  const int64_t N = B * S, p0 = (int64_t)blockIdx.x * 64, d0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  if (threadIdx.x < 64) {
    const int64_t p = p0 + tx;
    int64_t id = p < N ? ids[id_of(p, B, S, rows)] : -1;
    const bool held = id >= 0 && id < V;
    if (p < N && !held && oob && blockIdx.y == 0) atomicAdd(oob, 1);
    tok[tx] = held ? id : -1;
  }
  __syncthreads();
  float v[16];
  const int64_t d = d0 + tx;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int64_t id = tok[ty + 4 * u];
    v[u] = d < D && id >= 0 ? scale * Wt[d + D * id] : 0.f;
  }
#pragma unroll
  for (int u = 0; u < 16; ++u) tile[ty + 4 * u][tx] = v[u];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int j = ty + 4 * u;
    if (p0 + tx < N && d0 + j < D) out[p0 + tx + N * (d0 + j)] = tile[tx][j];
  }
}

// ------------------------------------------------------------------ gradient
// 1. Every id finds its place among the sorted ones (its rank: how many are
//    smaller, or equal and before it), while dY [N, D] is turned into dYt, a
//    row's features adjacent (leading dimension Dp, a multiple of 4).
// 2. The sorted rows are summed in chunks of kChunk, a wave each: a token
//    whose rows lie inside one chunk is written to the table, the sums of one
//    that goes on into the next chunk are kept.
// 3. Those are added in the order of the chunks.
// Ids outside the table sort last, as V, and are left out.  The order of every
// sum is fixed by the ids alone.
constexpr int kChunk = 16;

struct TokArgs {
  const int32_t* ids;
  const float* dY;
  float* gWt;
  int64_t B, S, V, D, N, Dp;
  int rows, accumulate;
  float scale;
  float* dYt;      // [N][Dp]
  int32_t* sid;    // [N] sorted ids
  int32_t* order;  // [N] their rows
  float* part;     // [chunks][2][Dp]
  int chunks;
};

__device__ __forceinline__ int32_t key_of(int32_t id, int64_t V) {
  return id >= 0 && id < V ? id : (int32_t)V;
}

// how many of ids[j0 .. j1) have a key below t
__device__ __forceinline__ int below(const int32_t* ids, int64_t V, int64_t j0, int64_t j1, int64_t t) {
  int n = 0;
  int64_t j = j0;
  for (; j + 16 <= j1; j += 16) {
    i32x4u x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const i32x4u*>(ids + j + 4 * u);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) n += key_of(x[u][e], V) < t;
  }
  for (; j < j1; ++j) n += key_of(ids[j], V) < t;
  return n;
}

__global__ void __launch_bounds__(256) token_sort_kernel(TokArgs a, int sort_blocks) {
  __shared__ float tile[64][65];
  if ((int)blockIdx.x < sort_blocks) {
    // 32 ids a block; the eight half-waves share the comparisons of each
    int* counts = reinterpret_cast<int*>(&tile[0][0]);  // [8][32]
    const int at = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t i0 = (int64_t)blockIdx.x * 32, i1 = i0 + 32 < a.N ? i0 + 32 : a.N;
    const int64_t i = i0 + at;
    const int32_t key = i < a.N ? key_of(a.ids[i], a.V) : 0;
    const int64_t per = (a.N + 7) / 8, j0 = part * per, j1 = j0 + per < a.N ? j0 + per : a.N;
    int n = 0;
    if (j0 < j1) {
      // before the block's ids an equal one counts, after them it does not
      const int64_t a1 = j1 < i0 ? j1 : i0, b0 = j0 > i1 ? j0 : i1;
      if (j0 < a1) n += below(a.ids, a.V, j0, a1, (int64_t)key + 1);
      if (b0 < j1) n += below(a.ids, a.V, b0, j1, key);
      for (int64_t j = j0 > i0 ? j0 : i0; j < (j1 < i1 ? j1 : i1); ++j) n += key_of(a.ids[j], a.V) < (int64_t)key + (j < i);
    }
    counts[part * 32 + at] = n;
    __syncthreads();
    if (part == 0 && i < a.N) {
      int rank = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) rank += counts[q * 32 + at];
      a.sid[rank] = key;
      a.order[rank] = (int32_t)row_of(i, a.B, a.S, a.rows);
    }
    return;
  }
  const int64_t t = (int64_t)blockIdx.x - sort_blocks, tiles = (a.N + 63) / 64;
  const int64_t p0 = t % tiles * 64, d0 = t / tiles * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int j = ty + 4 * u;
    tile[j][tx] = p0 + tx < a.N && d0 + j < a.D ? a.dY[p0 + tx + a.N * (d0 + j)] : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int64_t p = p0 + ty + 4 * u;
    if (p < a.N && d0 + tx < a.Dp) a.dYt[p * a.Dp + d0 + tx] = tile[tx][ty + 4 * u];
  }
}

// row v of the table, features d .. d + 3
__device__ __forceinline__ void put(const TokArgs& a, int64_t v, int64_t d, f32x4 x) {
  float* g = a.gWt + a.D * v + d;
  x *= a.scale;
  if (d + 4 <= a.D) {
    if (a.accumulate) x += *reinterpret_cast<const f32x4u*>(g);
    *reinterpret_cast<f32x4u*>(g) = x;
  } else {
    for (int e = 0; e < 4; ++e)
      if (d + e < a.D) g[e] = a.accumulate ? g[e] + x[e] : x[e];
  }
}

// blocks [0, zero_blocks): zeros for the table's rows that no id names, a wave
// for 64 rows; then a wave for each chunk and 256 features.
__global__ void __launch_bounds__(256) token_sum_kernel(TokArgs a, int zero_blocks, int cols) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < zero_blocks) {
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * 64;
    if (v0 >= a.V) return;
    const int64_t v = v0 + lane;
    int64_t lo = 0, hi = a.N;  // first sorted id that is not below v
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (a.sid[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    uint64_t unused = __ballot(v < a.V && (lo == a.N || a.sid[lo] != v));
    while (unused) {
      const int u = __ffsll((unsigned long long)unused) - 1;
      unused &= unused - 1;
      float* g = a.gWt + a.D * (v0 + u);
      for (int64_t d = 4 * lane; d < a.D; d += 256) {
        if (d + 4 <= a.D) *reinterpret_cast<f32x4u*>(g + d) = f32x4{0.f, 0.f, 0.f, 0.f};
        else
          for (int e = 0; e < 4; ++e)
            if (d + e < a.D) g[d + e] = 0.f;
      }
    }
    return;
  }
  const int64_t w = ((int64_t)blockIdx.x - zero_blocks) * 4 + wave;
  const int c = (int)(w / cols);
  if (c >= a.chunks) return;
  const int64_t d = (w % cols) * 256 + 4 * lane;
  const int64_t first = (int64_t)c * kChunk;
  // lanes 0 .. kChunk + 1: the ids of entries first - 1 .. first + kChunk
  const int64_t e = first - 1 + lane;
  const bool in = lane < kChunk + 2 && e >= 0 && e < a.N;
  const int my_id = in ? a.sid[e] : -1;
  const int my_row = in && e >= first ? a.order[e] : 0;
  int id[kChunk + 2];
#pragma unroll
  for (int i = 0; i < kChunk + 2; ++i) id[i] = __builtin_amdgcn_readlane(my_id, i);
  f32x4 x[kChunk];
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const int64_t row = __builtin_amdgcn_readlane(my_row, i + 1);
    x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (id[i + 1] >= 0 && id[i + 1] < a.V && d < a.Dp) x[i] = *reinterpret_cast<const f32x4*>(a.dYt + row * a.Dp + d);
  }
  bool begun = id[0] != id[1];  // the token's first row is in this chunk
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    if (id[i + 1] < 0 || id[i + 1] >= a.V) return;  // past the last
    s += x[i];
    const bool ends = id[i + 2] != id[i + 1];
    if (!ends && i + 1 < kChunk) continue;
    if (d < a.Dp) {
      if (begun && ends) put(a, id[i + 1], d, s);
      else *reinterpret_cast<f32x4*>(a.part + ((int64_t)c * 2 + begun) * a.Dp + d) = s;
    }
    begun = true;
    s = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// A block for each chunk and 256 features: where a token begins in the chunk
// and goes on, its kept sums in order.
__global__ void __launch_bounds__(64) token_join_kernel(TokArgs a) {
  const int c = (int)blockIdx.x;
  const int64_t last = (int64_t)(c + 1) * kChunk - 1;
  if (last + 1 >= a.N) return;
  const int32_t v = a.sid[last];
  if (v >= a.V || a.sid[last + 1] != v) return;
  if (last >= kChunk && a.sid[last - kChunk] == v) return;  // it began before this chunk
  int64_t lo = last + 1, hi = a.N;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (a.sid[mid] <= v) lo = mid + 1;
    else hi = mid;
  }
  const int end = (int)((lo - 1) / kChunk);
  const int64_t d = (int64_t)blockIdx.y * 256 + 4 * threadIdx.x;
  if (d >= a.Dp) return;
  f32x4 s = *reinterpret_cast<const f32x4*>(a.part + ((int64_t)c * 2 + 1) * a.Dp + d);
#pragma unroll 8
  for (int q = c + 1; q <= end; ++q) s += *reinterpret_cast<const f32x4*>(a.part + (int64_t)q * 2 * a.Dp + d);
  put(a, v, d, s);
}

int check_args(const char* who, int64_t B, int64_t S, int64_t V, int64_t D, float scale, int rows) {
  CNHIP_REQUIRE(B > 0 && S > 0 && V > 0 && D > 0, "%s: bad shape B=%lld S=%lld V=%lld D=%lld", who, (long long)B,
                (long long)S, (long long)V, (long long)D);
  CNHIP_REQUIRE(rows == CNHIP_ROWS_REF || rows == CNHIP_ROWS_BY_SAMPLE, "%s: bad row order %d", who, rows);
  CNHIP_REQUIRE(std::isfinite(scale), "%s: scale is not finite", who);
  CNHIP_REQUIRE(V < ((int64_t)1 << 31) && B < ((int64_t)1 << 30) && S < ((int64_t)1 << 30) &&
                    B * S < ((int64_t)1 << 30),
                "%s: too many ids or rows", who);
  CNHIP_REQUIRE(D <= 64 * 65535, "%s: embed_dim too large", who);
  return CNHIP_OK;
}

}  // namespace
}  // namespace cnhip

using cnhip::as_stream;

extern "C" {

int cnhip_token_embedding_forward(const int32_t* ids, const float* Wt, float* out, int64_t B, int64_t S, int64_t V,
                                  int64_t D, float scale, int32_t* oob_count, int rows, cnhip_stream_t stream) {
  const char* who = "cnhip_token_embedding_forward";
  CNHIP_TRY(cnhip::check_args(who, B, S, V, D, scale, rows));
  CNHIP_REQUIRE(ids && Wt && out, "%s: NULL pointer", who);
  const int64_t N = B * S;
  cnhip::HbmTimer timer("token_fwd_kernel", 4.0 * (double)N + 8.0 * (double)N * (double)D, as_stream(stream));
  hipLaunchKernelGGL(cnhip::token_fwd_kernel, dim3((unsigned)((N + 63) / 64), (unsigned)((D + 63) / 64)), dim3(256), 0,
                     as_stream(stream), ids, Wt, out, B, S, V, D, scale, rows, oob_count);
  return cnhip::check_launch(who);
}

int cnhip_token_embedding_backward(const int32_t* ids, const float* dY, float* gWt, int64_t B, int64_t S, int64_t V,
                                   int64_t D, float scale, int accumulate, int rows, cnhip_stream_t stream) {
  const char* who = "cnhip_token_embedding_backward";
  CNHIP_TRY(cnhip::check_args(who, B, S, V, D, scale, rows));
  CNHIP_REQUIRE(ids && dY && gWt, "%s: NULL pointer", who);
  CNHIP_REQUIRE(accumulate == 0 || accumulate == 1, "%s: accumulate must be 0 or 1", who);
  hipStream_t st = as_stream(stream);
  cnhip::TokArgs a{};
  a.ids = ids;
  a.dY = dY;
  a.gWt = gWt;
  a.B = B;
  a.S = S;
  a.V = V;
  a.D = D;
  a.N = B * S;
  a.Dp = (D + 3) / 4 * 4;
  a.rows = rows;
  a.accumulate = accumulate;
  a.scale = scale;
  a.chunks = (int)((a.N + cnhip::kChunk - 1) / cnhip::kChunk);
  const int64_t tiles = (a.N + 63) / 64 * ((D + 63) / 64), sort_blocks = (a.N + 31) / 32;
  const int cols = (int)((a.Dp + 255) / 256);
  const int64_t zero_blocks = accumulate ? 0 : (V + 255) / 256, sum_blocks = ((int64_t)a.chunks * cols + 3) / 4;
  CNHIP_REQUIRE(tiles + sort_blocks < ((int64_t)1 << 31) && zero_blocks + sum_blocks < ((int64_t)1 << 31),
                "%s: too large", who);
  const size_t rows_bytes = (size_t)(a.N * a.Dp) * sizeof(float);
  const size_t part_bytes = (size_t)a.chunks * 2 * (size_t)a.Dp * sizeof(float);
  const size_t ints = (size_t)a.N * sizeof(int32_t);
  void* ws = nullptr;
  CNHIP_TRY(cnhip::scratch(st, cnhip::kScratchLayer, rows_bytes + part_bytes + 2 * ints, &ws, who));
  a.dYt = static_cast<float*>(ws);
  a.part = a.dYt + a.N * a.Dp;
  a.sid = reinterpret_cast<int32_t*>(a.part + (int64_t)a.chunks * 2 * a.Dp);
  a.order = a.sid + a.N;
  hipLaunchKernelGGL(cnhip::token_sort_kernel, dim3((unsigned)(sort_blocks + tiles)), dim3(256), 0, st, a,
                     (int)sort_blocks);
  CNHIP_TRY(cnhip::check_launch(who));
  {
    // every row's gradient read once, every row of the table that is written
    cnhip::HbmTimer timer("token_sum_kernel",
                          4.0 * (double)a.N * (double)D + (accumulate ? 8.0 * (double)a.N : 4.0 * (double)V) * (double)D, st);
    hipLaunchKernelGGL(cnhip::token_sum_kernel, dim3((unsigned)(zero_blocks + sum_blocks)), dim3(256), 0, st, a,
                       (int)zero_blocks, cols);
    CNHIP_TRY(cnhip::check_launch(who));
  }
  hipLaunchKernelGGL(cnhip::token_join_kernel, dim3((unsigned)a.chunks, (unsigned)cols), dim3(64), 0, st, a);
  return cnhip::check_launch(who);
}

}  // extern "C"
