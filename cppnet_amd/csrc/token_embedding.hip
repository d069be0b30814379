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

// Row of the sequence that the id at j = b + B s belongs to, and the reverse.
__device__ __forceinline__ int64_t row_of(int64_t j, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? j : j / B + S * (j % B);
}
__device__ __forceinline__ int64_t id_of(int64_t p, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? p : p / S + B * (p % S);
}

// A 64 x 64 tile turned through LDS, float4s along either side: element c of
// row r lies at tile[r][lane_of(r, c)], which spreads both the rows' float4s and
// the single elements of a column over all banks.
constexpr int TS = 64;
__device__ __forceinline__ int lane_of(int r, int c) { return c ^ (r & 60); }

// Four floats from p, of which the first n exist (zeros for the others).
__device__ __forceinline__ f32x4 get4(const float* p, int64_t n) {
  if (n >= 4) return *reinterpret_cast<const f32x4u*>(p);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) x[e] = p[e];
  return x;
}
__device__ __forceinline__ void put4(float* p, int64_t n, f32x4 x) {
  if (n >= 4) {
    *reinterpret_cast<f32x4u*>(p) = x;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) p[e] = x[e];
}

// 64 rows x 64 features: read along the features of the table, turned, written
// along the rows of out.  Bound by memory: 14329 rows of 1000 28 us (115 MB, 4.1
// TB/s).
__global__ void __launch_bounds__(256) token_fwd_kernel(const int32_t* __restrict__ ids, const float* __restrict__ Wt,
                                                        float* __restrict__ out, int64_t B, int64_t S, int64_t V,
                                                        int64_t D, float scale, int rows, int32_t* __restrict__ oob) {
  __shared__ __align__(16) float tile[64][TS];  // [feature][row]
  __shared__ int32_t tok[64];
  const int64_t N = B * S, p0 = (int64_t)blockIdx.x * 64, d0 = (int64_t)blockIdx.y * 64;
  if (threadIdx.x < 64) {
    const int64_t p = p0 + threadIdx.x;
    const int32_t id = p < N ? ids[id_of(p, B, S, rows)] : -1;
    const bool held = id >= 0 && id < V;
    if (p < N && !held && oob && blockIdx.y == 0) atomicAdd(oob, 1);
    tok[threadIdx.x] = held ? id : -1;
  }
  __syncthreads();
  const int four = 4 * (threadIdx.x & 15), one = threadIdx.x >> 4;
  f32x4 x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int32_t id = tok[one + 16 * u];
    x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (id >= 0) x[u] = get4(Wt + D * (int64_t)id + d0 + four, D - d0 - four);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[four + e][lane_of(four + e, one + 16 * u)] = scale * x[u][e];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = one + 16 * u;
    if (d0 + d < D) put4(out + p0 + four + N * (d0 + d), N - p0 - four, *reinterpret_cast<const f32x4*>(&tile[d][lane_of(d, four)]));
  }
}

// ------------------------------------------------------------------ gradient
// 1. The ids are sorted, equal ones in their order (each finds how many are
//    smaller, or equal and before it; very many by a radix sort), while dY
//    [N, D] is turned into dYt, a row's features adjacent (leading dimension
//    Dp, a multiple of 4), and the table's rows that no id names get zeros.
// 2. The sorted rows are summed in chunks of kChunk, a wave each: a token
//    whose rows lie inside one chunk is written to the table, the sums of one
//    that goes on into the next chunk are kept.
// 3. Those are added in the order of the chunks.
// Ids outside the table sort last, as V, and are left out.  The order of every
// sum is fixed by the ids alone.
// Bound by memory: 14329 rows of 1000, table of 50001: the first launch 76 us (200
// MB of zeros, 115 MB of turning, the sort beside them; 4.1 TB/s), the sums 17, their
// joining 8.
constexpr int kChunk = 16;

constexpr int64_t kRankMost = 24576;

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

// Up to kRankMost ids are sorted by comparing each with every other: 2 N^2
// instructions over all lanes, beside the turning of dY in the same launch.
// More take a radix sort in launches of its own.  The whole gradient at width
// 512 and 32000 ids, comparing against radix sort: 8192 rows 40 and 79 us,
// 16384 58 and 85, 24576 86 and 90, 32768 125 and 99.
constexpr int kIdChunk = 8192;  // ids in LDS at a time

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kSortIds = 16;                // ids a block
constexpr int kSortParts = 256 / kSortIds;  // threads that share an id's comparisons

// how many of this thread's fours of keys in [q0, q1) are below t
__device__ __forceinline__ int below(const i32x4* keys, int q0, int q1, int part, int32_t t) {
  int n = 0;
#pragma unroll 8
  for (int q = q0 + part; q < q1; q += kSortParts) {
    const i32x4 x = keys[q];
#pragma unroll
    for (int e = 0; e < 4; ++e) n += x[e] < t;
  }
  return n;
}

// Turns tile t of dY into dYt.
__device__ __forceinline__ void turn_tile(const TokArgs& a, int64_t t, float (*tile)[TS]) {
  const int64_t tiles = (a.N + 63) / 64, p0 = t % tiles * 64, d0 = t / tiles * 64;
  const int four = 4 * (threadIdx.x & 15), one = threadIdx.x >> 4;
  f32x4 x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t d = d0 + one + 16 * u;
    x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (d < a.D) x[u] = get4(a.dY + p0 + four + a.N * d, a.N - p0 - four);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[four + e][lane_of(four + e, one + 16 * u)] = x[u][e];  // [row][feature]
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t p = p0 + one + 16 * u;
    if (p < a.N && d0 + four < a.Dp)
      *reinterpret_cast<f32x4*>(a.dYt + p * a.Dp + d0 + four) = *reinterpret_cast<const f32x4*>(&tile[one + 16 * u][lane_of(one + 16 * u, four)]);
  }
}

// Zeros for those of a block's rows of the table that no id names.  The block
// reads all ids; where they are many it takes more rows.
__host__ __device__ __forceinline__ int zero_rows(int64_t N) {
  return N <= 131072 ? 64 : N <= 1048576 ? 512 : 4096;
}

__device__ __forceinline__ void zero_unused(const TokArgs& a, int64_t blk, unsigned char* used) {
  const int rows = zero_rows(a.N), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t v0 = blk * rows;
  for (int r = 4 * threadIdx.x; r < rows; r += 1024) *reinterpret_cast<uint32_t*>(used + r) = 0;
  __syncthreads();
  int64_t j = 4 * threadIdx.x;
#pragma unroll 8
  for (; j + 4 <= a.N; j += 1024) {
    const i32x4 x = *reinterpret_cast<const i32x4u*>(a.ids + j);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (x[e] >= v0 && x[e] < v0 + rows) used[x[e] - v0] = 1;
  }
  for (; j < a.N; ++j)
    if (a.ids[j] >= v0 && a.ids[j] < v0 + rows) used[a.ids[j] - v0] = 1;
  __syncthreads();
  for (int r = wave; r < rows && v0 + r < a.V; r += 4) {
    if (used[r]) continue;
    float* g = a.gWt + a.D * (v0 + r);
    for (int64_t d = 4 * lane; d < a.D; d += 256) put4(g + d, a.D - d, f32x4{0.f, 0.f, 0.f, 0.f});
  }
}

__global__ void __launch_bounds__(256) token_sort_kernel(TokArgs a, int sort_blocks, int zero_blocks) {
  __shared__ __align__(16) int32_t lds[kIdChunk];  // ids, or a tile of dY
  static_assert(sizeof(lds) >= 64 * TS * sizeof(float), "a tile fits");
  if ((int)blockIdx.x >= sort_blocks) {
    const int64_t blk = (int64_t)blockIdx.x - sort_blocks;
    if (blk < zero_blocks) zero_unused(a, blk, reinterpret_cast<unsigned char*>(lds));
    else turn_tile(a, blk - zero_blocks, reinterpret_cast<float (*)[TS]>(lds));
    return;
  }
  const int at = threadIdx.x % kSortIds, part = threadIdx.x / kSortIds;
  const int N = (int)a.N, i0 = (int)blockIdx.x * kSortIds, i = i0 + at;
  const int32_t key = i < N ? key_of(a.ids[i], a.V) : 0;
  int n = 0;
  for (int c0 = 0; c0 < N; c0 += kIdChunk) {
    const int m = N - c0 < kIdChunk ? N - c0 : kIdChunk, m4 = (m + 3) / 4 * 4;
    __syncthreads();
#pragma unroll 8
    for (int j = 4 * threadIdx.x; j < m4; j += 1024) {
      i32x4 x;
      if (j + 4 <= m) {
        x = *reinterpret_cast<const i32x4u*>(a.ids + c0 + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = key_of(x[e], a.V);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = j + e < m ? key_of(a.ids[c0 + j + e], a.V) : INT32_MAX;
      }
      *reinterpret_cast<i32x4*>(lds + j) = x;
    }
    __syncthreads();
    // before the block's ids an equal one counts, after them it does not
    const int lo = min(max(i0 - c0, 0), m4), hi = min(max(i0 + kSortIds - c0, 0), m4);
    const i32x4* fours = reinterpret_cast<const i32x4*>(lds);
    n += below(fours, 0, lo / 4, part, key + 1);  // key + 1 <= V + 1 <= INT32_MAX
    n += below(fours, hi / 4, m4 / 4, part, key);
    if (lo + part < hi) n += lds[lo + part] < key + (c0 + lo + part < i);
  }
  __syncthreads();
  lds[part * kSortIds + at] = n;
  __syncthreads();
  if (part == 0 && i < N) {
    int rank = 0;
#pragma unroll
    for (int q = 0; q < kSortParts; ++q) rank += lds[q * kSortIds + at];
    a.sid[rank] = key;
    a.order[rank] = (int32_t)row_of(i, a.B, a.S, a.rows);
  }
}

// The radix sort: eight bits a pass, from the lowest; a block counts, then
// moves, kRadixTile keys, each of its four waves a run of them, 64 at a time,
// so equal digits keep their order.
constexpr int kRadixTile = 4096;

struct RadixArgs {
  const int32_t *key_in, *row_in;  // null in the first pass: the ids and their rows
  int32_t *key_out, *row_out;
  int32_t* counts;                 // [256][blocks], then their exclusive sums
  int shift, blocks;
};

__device__ __forceinline__ int32_t radix_key(const TokArgs& a, const RadixArgs& r, int64_t i) {
  return r.key_in ? r.key_in[i] : key_of(a.ids[i], a.V);
}

__global__ void __launch_bounds__(256) token_radix_count_kernel(TokArgs a, RadixArgs r, int zero_blocks, int turn_blocks) {
  __shared__ __align__(16) float tile[64][TS];
  if ((int)blockIdx.x < zero_blocks + turn_blocks) {  // in the first pass
    if ((int)blockIdx.x < zero_blocks) zero_unused(a, blockIdx.x, reinterpret_cast<unsigned char*>(tile));
    else turn_tile(a, (int64_t)blockIdx.x - zero_blocks, tile);
    return;
  }
  int32_t* hist = reinterpret_cast<int32_t*>(tile);
  const int blk = (int)blockIdx.x - zero_blocks - turn_blocks;
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blk * kRadixTile;
  for (int j = threadIdx.x; j < kRadixTile; j += 256)
    if (i0 + j < a.N) atomicAdd(&hist[radix_key(a, r, i0 + j) >> r.shift & 255], 1);
  __syncthreads();
  r.counts[(int64_t)threadIdx.x * r.blocks + blk] = hist[threadIdx.x];
}

// exclusive sums over counts in place (one block)
__global__ void __launch_bounds__(1024) token_radix_scan_kernel(RadixArgs r) {
  __shared__ int32_t wave_sum[16];
  const int64_t total = (int64_t)256 * r.blocks, per = (total + 1023) / 1024;
  const int64_t lo = min(total, (int64_t)threadIdx.x * per), hi = min(total, lo + per);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t s = 0;
#pragma unroll 8
  for (int64_t i = lo; i < hi; ++i) s += r.counts[i];
  int32_t x = s;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) wave_sum[wave] = x;
  __syncthreads();
  int32_t run = x - s;
  for (int w = 0; w < wave; ++w) run += wave_sum[w];
  for (int64_t i = lo; i < hi; ++i) {
    const int32_t c = r.counts[i];
    r.counts[i] = run;
    run += c;
  }
}

__global__ void __launch_bounds__(256) token_radix_move_kernel(TokArgs a, RadixArgs r) {
  __shared__ int32_t at[4][256];  // where a wave's next key of a digit goes
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)blockIdx.x * kRadixTile + wave * (kRadixTile / 4);
  for (int w = 0; w < 4; ++w) at[w][threadIdx.x] = 0;
  __syncthreads();
  for (int j = lane; j < kRadixTile / 4; j += 64)
    if (i0 + j < a.N) atomicAdd(&at[wave][radix_key(a, r, i0 + j) >> r.shift & 255], 1);
  __syncthreads();
  {
    int32_t run = r.counts[(int64_t)threadIdx.x * r.blocks + blockIdx.x];
    for (int w = 0; w < 4; ++w) {
      const int32_t c = at[w][threadIdx.x];
      at[w][threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int j = 0; j < kRadixTile / 4; j += 64) {
    const int64_t i = i0 + j + lane;
    const bool in = i < a.N;
    const int32_t key = in ? radix_key(a, r, i) : 0;
    const int digit = key >> r.shift & 255;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t set = __ballot(digit >> b & 1);
      same &= digit >> b & 1 ? set : ~set;
    }
    const int before = __popcll(same & (((uint64_t)1 << lane) - 1));
    const int32_t base = at[wave][digit];
    // every lane has its digit's place before the first of them moves it on
    __builtin_amdgcn_wave_barrier();
    if (in && before == 0) at[wave][digit] = base + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) {
      r.key_out[base + before] = key;
      r.row_out[base + before] = r.row_in ? r.row_in[i] : (int32_t)row_of(i, a.B, a.S, a.rows);
    }
  }
}

// row v of the table, features d .. d + 3
__device__ __forceinline__ void put(const TokArgs& a, int64_t v, int64_t d, f32x4 x) {
  float* g = a.gWt + a.D * v + d;
  x *= a.scale;
  if (a.accumulate) x += get4(g, a.D - d);
  put4(g, a.D - d, x);
}

// A wave for each chunk and 256 features.
__global__ void __launch_bounds__(256) token_sum_kernel(TokArgs a, int cols) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t w = (int64_t)blockIdx.x * 4 + wave;
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
  // the chunk it ends in: the first whose next entry is another's, 64 at a time
  int end = c + 1;
  for (;; end += 64) {
    const int64_t next = ((int64_t)end + threadIdx.x + 1) * kChunk;
    const uint64_t ends = __ballot(next >= a.N || a.sid[next] != v);
    if (!ends) continue;
    end += __ffsll((unsigned long long)ends) - 1;
    break;
  }
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
  CNHIP_REQUIRE(V < ((int64_t)1 << 31) - 1 && B < ((int64_t)1 << 30) && S < ((int64_t)1 << 30) &&
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
  const int64_t tiles = (a.N + 63) / 64 * ((D + 63) / 64);
  const bool radix = a.N > cnhip::kRankMost;
  const int64_t sort_blocks = radix ? (a.N + cnhip::kRadixTile - 1) / cnhip::kRadixTile
                                    : (a.N + cnhip::kSortIds - 1) / cnhip::kSortIds;
  const int cols = (int)((a.Dp + 255) / 256);
  const int zr = cnhip::zero_rows(a.N);
  const int64_t zero_blocks = accumulate ? 0 : (V + zr - 1) / zr, sum_blocks = ((int64_t)a.chunks * cols + 3) / 4;
  CNHIP_REQUIRE(tiles + sort_blocks + zero_blocks < ((int64_t)1 << 31) && sum_blocks < ((int64_t)1 << 31),
                "%s: too large", who);
  const size_t rows_bytes = (size_t)(a.N * a.Dp) * sizeof(float);
  const size_t part_bytes = (size_t)a.chunks * 2 * (size_t)a.Dp * sizeof(float);
  const size_t ints = (size_t)a.N * sizeof(int32_t), counts = (size_t)sort_blocks * 256 * sizeof(int32_t);
  void* ws = nullptr;
  CNHIP_TRY(cnhip::scratch(st, cnhip::kScratchLayer, rows_bytes + part_bytes + (radix ? 4 * ints + counts : 2 * ints), &ws,
                           who));
  a.dYt = static_cast<float*>(ws);
  a.part = a.dYt + a.N * a.Dp;
  a.sid = reinterpret_cast<int32_t*>(a.part + (int64_t)a.chunks * 2 * a.Dp);
  a.order = a.sid + a.N;
  if (!radix) {
    hipLaunchKernelGGL(cnhip::token_sort_kernel, dim3((unsigned)(sort_blocks + zero_blocks + tiles)), dim3(256), 0, st, a,
                       (int)sort_blocks, (int)zero_blocks);
    CNHIP_TRY(cnhip::check_launch(who));
  } else {
    int bits = 1;
    while (((int64_t)1 << bits) <= V) ++bits;  // keys are 0 .. V
    const int passes = (bits + 7) / 8;
    int32_t* pair[2][2] = {{a.sid, a.order}, {a.order + a.N, a.order + 2 * a.N}};
    cnhip::RadixArgs r{nullptr, nullptr, nullptr, nullptr, a.order + 3 * a.N, 0, (int)sort_blocks};
    for (int pass = 0; pass < passes; ++pass) {
      int32_t** to = pair[(passes - 1 - pass) & 1];  // the last pass ends in sid and order
      r.key_out = to[0];
      r.row_out = to[1];
      r.shift = 8 * pass;
      const int64_t zero = pass == 0 ? zero_blocks : 0, turn = pass == 0 ? tiles : 0;
      hipLaunchKernelGGL(cnhip::token_radix_count_kernel, dim3((unsigned)(zero + turn + sort_blocks)), dim3(256), 0, st,
                         a, r, (int)zero, (int)turn);
      CNHIP_TRY(cnhip::check_launch(who));
      hipLaunchKernelGGL(cnhip::token_radix_scan_kernel, dim3(1), dim3(1024), 0, st, r);
      CNHIP_TRY(cnhip::check_launch(who));
      hipLaunchKernelGGL(cnhip::token_radix_move_kernel, dim3((unsigned)sort_blocks), dim3(256), 0, st, a, r);
      CNHIP_TRY(cnhip::check_launch(who));
      r.key_in = to[0];
      r.row_in = to[1];
    }
  }
  {
    // every row's gradient read once, every row of the table that is written
    cnhip::HbmTimer timer("token_sum_kernel",
                          4.0 * (double)a.N * (double)D + (accumulate ? 8.0 * (double)a.N : 4.0 * (double)V) * (double)D, st);
    hipLaunchKernelGGL(cnhip::token_sum_kernel, dim3((unsigned)sum_blocks), dim3(256), 0, st, a, cols);
    CNHIP_TRY(cnhip::check_launch(who));
  }
  hipLaunchKernelGGL(cnhip::token_join_kernel, dim3((unsigned)a.chunks, (unsigned)cols), dim3(64), 0, st, a);
  return cnhip::check_launch(who);
}

}  // extern "C"
