// Multi-head attention that keeps no probabilities: forward with the row
// log-sum-exp, and the backward that forms the probabilities again from it.
//
//   S = scale q k^T over the keys a query reads,  lse_i = log sum_j exp(S_ij),
//   P_ij = exp(S_ij - lse_i),  out = P v;
//   delta_i = sum_d dout_id out_id,  dS = P (dout v^T - delta) scale,
//   dq = dS k,  dk = dS^T q,  dv = P^T dout   (dk, dv summed over the query
//   heads that share a key head).
//
// The products run on fp32 MFMAs (v_mfma_f32_32x32x2f32) whose accumulators
// feed the next product without leaving the registers.  An accumulator holds
// for its column (lane & 31) the rows 8 (r / 4) + 4 (lane / 32) + r % 4, and a
// B operand holds for its column one k per half-wave: register r of a score
// tile is the B operand of the k pair {8 (r / 4) + r % 4, the same + 4}.  So the
// scores are formed with the contraction of the product that follows along
// their rows: S^T = k q^T for out and dq (keys along the rows, a query per
// lane, whose maximum, sum and rescaling are the lane's own), S = q k^T for dk
// and dv (queries along the rows, a key per lane).  The features of a row lie
// a whole column apart in memory, so a [feature][row] tile in LDS is staged
// with float4s along the rows as it stands, and serves both as the operand
// whose lanes are rows (one float per lane) and as the one whose lanes are
// features (four rows per float4).
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace cnhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// One [B*S, heads*dh] sequence: element (sample b, step s, column f) at
// p[b * sample + s * row + f * col].
template <class T>
struct Seq {
  T* p;
  int64_t sample, row, col;
  __device__ __forceinline__ T* at(int64_t b, int64_t s, int64_t f) const { return p + b * sample + s * row + f * col; }
};

struct AttArgs {
  Seq<const float> q, k, v, o, dout;
  Seq<float> out, dq, dk, dv;
  float* lse;              // [B*Sq, heads] in the row order of q, or null
  const float* lse_in;
  int64_t lse_sample, lse_row, lse_col;
  float* delta;            // [B][heads][Sq]
  int B, Sq, Sk, heads, kv_heads, dh;
  int group;               // query heads per key head
  float scale;
  int causal;
  const int32_t *k_len, *q_start;
};

// Keys of sample b, and the position of its first query.
__device__ __forceinline__ int keys_of(const AttArgs& a, int b) {
  return a.k_len ? min(max(a.k_len[b], 0), a.Sk) : a.Sk;
}
__device__ __forceinline__ int64_t start_of(const AttArgs& a, int b) {
  return a.q_start ? (int64_t)a.q_start[b] : (int64_t)a.Sk - a.Sq;
}
// Keys that query i reads: the first limit(..) of the sample's n.
__device__ __forceinline__ int limit(const AttArgs& a, int n, int64_t start, int64_t i) {
  if (!a.causal) return n;
  const int64_t l = start + i + 1;
  return (int)(l < 0 ? 0 : l < n ? l : n);
}

constexpr int RT = 32;       // rows of a streamed tile
constexpr int LS = RT + 4;   // floats between features of a tile in LDS
constexpr int NT = 256;      // threads of a block: four waves of 32 rows each

// A [DHP][RT] tile on its way to LDS: RT rows from `row0` on, of which
// `valid` exist; others, and features past dh, become zeros.
template <int DHP, bool UNIT>
struct TileLoad {
  static constexpr int U = DHP / 32;  // float4s per thread
  f32x4 v[U];
  __device__ __forceinline__ void load(const float* base, int64_t row, int64_t col, int valid, int dh) {
    const int r = 4 * ((int)threadIdx.x & 7), d0 = (int)threadIdx.x >> 3;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = d0 + 32 * u;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (d < dh) {
        const float* p = base + r * row + d * col;
        if (UNIT && r + 3 < valid) {
          x = *reinterpret_cast<const f32x4u*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (r + e < valid) x[e] = p[e * row];
        }
      }
      v[u] = x;
    }
  }
  __device__ __forceinline__ void store(float* lds) const {
    const int r = 4 * ((int)threadIdx.x & 7), d0 = (int)threadIdx.x >> 3;
#pragma unroll
    for (int u = 0; u < U; ++u) *reinterpret_cast<f32x4*>(lds + (d0 + 32 * u) * LS + r) = v[u];
  }
};

// The operand of this lane's row for a contraction over the features: feature
// 2 s + lane / 32 in register s, zeros past dh or where there is no row.
template <int DHP>
__device__ __forceinline__ void load_row(const float* base, int64_t col, bool held, int dh, float (&x)[DHP / 2]) {
  const int h = ((int)threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DHP / 2; ++s) {
    const int d = 2 * s + h;
    x[s] = held && d < dh ? base[d * col] : 0.f;
  }
}

// acc (rows of the tile x rows of the lanes) = tile x^T over the features
template <int DHP>
__device__ __forceinline__ f32x16 dot_rows(const float* tile, const float (&x)[DHP / 2]) {
  const int lane = (int)threadIdx.x & 63;
  const float* p = tile + (lane >> 5) * LS + (lane & 31);
  f32x16 acc = {};
#pragma unroll
  for (int s = 0; s < DHP / 2; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(p[2 * s * LS], x[s], acc, 0, 0, 0);
  return acc;
}
// acc (features x rows of the lanes) += tile^T p over the rows of the tile
template <int DHP>
__device__ __forceinline__ void add_rows(const float* tile, const f32x16& p, f32x16 (&acc)[DHP / 32]) {
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < DHP / 32; ++i) {
    const float* t = tile + (32 * i + (lane & 31)) * LS + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(t + 8 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], p[4 * q + e], acc[i], 0, 0, 0);
    }
  }
}
// stores acc (features x rows of the lanes) * f into this lane's row
template <int DHP>
__device__ __forceinline__ void store_row(float* base, int64_t col, bool held, int dh, float f,
                                          const f32x16 (&acc)[DHP / 32]) {
  const int h = ((int)threadIdx.x & 63) >> 5;
  if (!held) return;
#pragma unroll
  for (int i = 0; i < DHP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * i + 8 * (r / 4) + 4 * h + r % 4;
      if (d < dh) base[d * col] = acc[i][r] * f;
    }
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// Forward.  A block owns 128 rows of a key head's queries: row g Sq + i is
// query i of the g-th of the query heads that share the key head, so a
// sequence's single queries fill a wave together.
template <int DHP, bool UNIT>
__global__ void __launch_bounds__(NT) att_fwd_kernel(AttArgs a) {
  __shared__ __align__(16) float lds[2][DHP * LS];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int64_t rows = (int64_t)a.group * a.Sq;
  const int64_t r = (int64_t)blockIdx.x * 128 + 32 * wave + (lane & 31);
  const bool held = r < rows;
  const int head = kh * a.group + (int)(held ? r / a.Sq : 0);
  const int64_t i = held ? r % a.Sq : 0;
  const int n = keys_of(a, b);
  const int lim = held ? limit(a, n, start_of(a, b), i) : 0;
  float q[DHP / 2];
  load_row<DHP>(a.q.at(b, i, (int64_t)head * a.dh), a.q.col, held, a.dh, q);
  __shared__ int most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  atomicMax(&most, lim);
  __syncthreads();
  const int end = most;
  const float c = a.scale * kLog2e;
  const float* kp = a.k.at(b, 0, (int64_t)kh * a.dh);
  const float* vp = a.v.at(b, 0, (int64_t)kh * a.dh);

  f32x16 o[DHP / 32] = {};
  float m = -INFINITY, l = 0.f;  // of t = scale log2(e) s: maximum and sum of 2^(t - m)
  TileLoad<DHP, UNIT> tk, tv;
  if (end > 0) {
    tk.load(kp, a.k.row, a.k.col, n, a.dh);
    tv.load(vp, a.v.row, a.v.col, n, a.dh);
  }
  for (int j0 = 0; j0 < end; j0 += RT) {
    __syncthreads();
    tk.store(lds[0]);
    tv.store(lds[1]);
    __syncthreads();
    if (j0 + RT < end) {
      tk.load(kp + (j0 + RT) * a.k.row, a.k.row, a.k.col, n - j0 - RT, a.dh);
      tv.load(vp + (j0 + RT) * a.v.row, a.v.row, a.v.col, n - j0 - RT, a.dh);
    }
    if (!__any(lim > j0)) continue;
    f32x16 s = dot_rows<DHP>(lds[0], q);
    float most_s = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = j0 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
      s[e] = j < lim ? s[e] * c : -INFINITY;
      most_s = fmaxf(most_s, s[e]);
    }
    const float mn = fmaxf(m, fmaxf(most_s, other_half(most_s)));
    const float base = mn == -INFINITY ? 0.f : mn;  // no key read yet: every 2^(-inf) is 0
    const float f = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(s[e] - base);
      sum += s[e];
    }
    l = l * f + sum;
    m = mn;
#pragma unroll
    for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] *= f;
    add_rows<DHP>(lds[1], s, o);
  }
  l += other_half(l);
  store_row<DHP>(a.out.at(b, i, (int64_t)head * a.dh), a.out.col, held, a.dh, lim > 0 ? 1.f / l : 0.f, o);
  if (a.lse && held && lane < 32)
    a.lse[b * a.lse_sample + i * a.lse_row + head * a.lse_col] = lim > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// delta[b][head][i] = sum_d dout out
__global__ void __launch_bounds__(NT) att_delta_kernel(AttArgs a) {
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int b = (int)blockIdx.y / a.heads, head = (int)blockIdx.y % a.heads;
  if (i >= a.Sq) return;
  const float* g = a.dout.at(b, i, (int64_t)head * a.dh);
  const float* o = a.o.at(b, i, (int64_t)head * a.dh);
  float s = 0.f;
  for (int d = 0; d < a.dh; ++d) s = fmaf(g[d * a.dout.col], o[d * a.o.col], s);
  a.delta[(int64_t)blockIdx.y * a.Sq + i] = s;
}

__device__ __forceinline__ float lse2_of(const AttArgs& a, int b, int head, int64_t i) {
  const float l = a.lse_in[b * a.lse_sample + i * a.lse_row + head * a.lse_col];
  return l == -INFINITY ? INFINITY : l * kLog2e;  // a row that reads no key: every 2^(t - inf) is 0
}

// dq: a block owns 128 rows as in the forward and streams keys and values.
template <int DHP, bool UNIT>
__global__ void __launch_bounds__(NT) att_dq_kernel(AttArgs a) {
  __shared__ __align__(16) float lds[2][DHP * LS];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int64_t rows = (int64_t)a.group * a.Sq;
  const int64_t r = (int64_t)blockIdx.x * 128 + 32 * wave + (lane & 31);
  const bool held = r < rows;
  const int head = kh * a.group + (int)(held ? r / a.Sq : 0);
  const int64_t i = held ? r % a.Sq : 0;
  const int n = keys_of(a, b);
  const int lim = held ? limit(a, n, start_of(a, b), i) : 0;
  float q[DHP / 2], g[DHP / 2];
  load_row<DHP>(a.q.at(b, i, (int64_t)head * a.dh), a.q.col, held, a.dh, q);
  load_row<DHP>(a.dout.at(b, i, (int64_t)head * a.dh), a.dout.col, held, a.dh, g);
  const float lse = held ? lse2_of(a, b, head, i) : INFINITY;
  const float delta = held ? a.delta[((int64_t)b * a.heads + head) * a.Sq + i] : 0.f;
  __shared__ int most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  atomicMax(&most, lim);
  __syncthreads();
  const int end = most;
  const float c = a.scale * kLog2e;
  const float* kp = a.k.at(b, 0, (int64_t)kh * a.dh);
  const float* vp = a.v.at(b, 0, (int64_t)kh * a.dh);
  f32x16 acc[DHP / 32] = {};
  TileLoad<DHP, UNIT> tk, tv;
  if (end > 0) {
    tk.load(kp, a.k.row, a.k.col, n, a.dh);
    tv.load(vp, a.v.row, a.v.col, n, a.dh);
  }
  for (int j0 = 0; j0 < end; j0 += RT) {
    __syncthreads();
    tk.store(lds[0]);
    tv.store(lds[1]);
    __syncthreads();
    if (j0 + RT < end) {
      tk.load(kp + (j0 + RT) * a.k.row, a.k.row, a.k.col, n - j0 - RT, a.dh);
      tv.load(vp + (j0 + RT) * a.v.row, a.v.row, a.v.col, n - j0 - RT, a.dh);
    }
    if (!__any(lim > j0)) continue;
    f32x16 s = dot_rows<DHP>(lds[0], q);
    const f32x16 dp = dot_rows<DHP>(lds[1], g);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = j0 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
      s[e] = j < lim ? __builtin_amdgcn_exp2f(fmaf(s[e], c, -lse)) * (dp[e] - delta) : 0.f;
    }
    add_rows<DHP>(lds[0], s, acc);
  }
  store_row<DHP>(a.dq.at(b, i, (int64_t)head * a.dh), a.dq.col, held, a.dh, a.scale, acc);
}

// dk, dv: a block owns 128 keys of a key head and streams the queries and
// output gradients of the heads that share it, one head after the other.
template <int DHP, bool UNIT>
__global__ void __launch_bounds__(NT) att_dkv_kernel(AttArgs a) {
  __shared__ __align__(16) float lds[2][DHP * LS];
  __shared__ __align__(16) float stat[2][RT];  // lse (base 2), delta of the tile's queries
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int key0 = (int)blockIdx.x * 128;
  const int key = key0 + 32 * wave + (lane & 31);
  const int n = keys_of(a, b);
  const int64_t start = start_of(a, b);
  const bool held = key < n;
  float k[DHP / 2], v[DHP / 2];
  const int at = key < a.Sk ? key : 0;
  load_row<DHP>(a.k.at(b, at, (int64_t)kh * a.dh), a.k.col, held, a.dh, k);
  load_row<DHP>(a.v.at(b, at, (int64_t)kh * a.dh), a.v.col, held, a.dh, v);
  const float c = a.scale * kLog2e;
  // the first query that reads the block's first key
  int64_t first = a.causal ? key0 - start : 0;
  first = first < 0 ? 0 : first / RT * RT;
  const int tiles = key0 < n && first < a.Sq ? (int)((a.Sq - first + RT - 1) / RT) : 0;
  f32x16 dk[DHP / 32] = {}, dv[DHP / 32] = {};
  TileLoad<DHP, UNIT> tq, tg;
  float st = 0.f;
  auto load = [&](int t) {
    const int head = kh * a.group + t / tiles;
    const int64_t i0 = first + (int64_t)(t % tiles) * RT;
    const int valid = (int)(a.Sq - i0 < RT ? a.Sq - i0 : RT);
    tq.load(a.q.at(b, i0, (int64_t)head * a.dh), a.q.row, a.q.col, valid, a.dh);
    tg.load(a.dout.at(b, i0, (int64_t)head * a.dh), a.dout.row, a.dout.col, valid, a.dh);
    const int r = (int)threadIdx.x & 31;
    if (threadIdx.x < RT) st = r < valid ? lse2_of(a, b, head, i0 + r) : INFINITY;
    else if (threadIdx.x < 2 * RT) st = r < valid ? a.delta[((int64_t)b * a.heads + head) * a.Sq + i0 + r] : 0.f;
  };
  const int total = tiles * a.group;
  if (total > 0) load(0);
  for (int t = 0; t < total; ++t) {
    __syncthreads();
    tq.store(lds[0]);
    tg.store(lds[1]);
    if (threadIdx.x < 2 * RT) stat[threadIdx.x / RT][threadIdx.x & 31] = st;
    __syncthreads();
    if (t + 1 < total) load(t + 1);
    const int64_t i0 = first + (int64_t)(t % tiles) * RT;
    if (a.causal && start + i0 + RT - 1 < key0 + 32 * wave) continue;  // no query of the tile reads this wave's keys
    f32x16 s = dot_rows<DHP>(lds[0], k);
    f32x16 dp = dot_rows<DHP>(lds[1], v);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = 8 * q + 4 * (lane >> 5);
      const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[0][r]);
      const f32x4 delta = *reinterpret_cast<const f32x4*>(&stat[1][r]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool reads = held && (!a.causal || key <= start + i0 + r + e);
        s[4 * q + e] = reads ? __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], c, -lse[e])) : 0.f;
        dp[4 * q + e] = s[4 * q + e] * (dp[4 * q + e] - delta[e]);
      }
    }
    add_rows<DHP>(lds[1], s, dv);
    add_rows<DHP>(lds[0], dp, dk);
  }
  // keys past the sample's last are nobody's: their gradients are zeros
  const bool stored = key < a.Sk;
  store_row<DHP>(a.dk.at(b, at, (int64_t)kh * a.dh), a.dk.col, stored, a.dh, a.scale, dk);
  store_row<DHP>(a.dv.at(b, at, (int64_t)kh * a.dh), a.dv.col, stored, a.dh, 1.f, dv);
}

constexpr int kMaxHeadDim = 128;

template <class T>
Seq<T> seq(T* p, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? Seq<T>{p, 1, B, B * S} : Seq<T>{p, S, 1, B * S};
}

// f(the kernel's feature padding as an integral constant, whether a step's
// neighbours are adjacent)
template <class F>
void dispatch(int dh, bool unit, F&& f) {
  auto by = [&](auto d) {
    if (unit) f(d, std::true_type{});
    else f(d, std::false_type{});
  };
  if (dh <= 32) by(std::integral_constant<int, 32>{});
  else if (dh <= 64) by(std::integral_constant<int, 64>{});
  else if (dh <= 96) by(std::integral_constant<int, 96>{});
  else by(std::integral_constant<int, 128>{});
}

int check_args(const char* who, int64_t B, int64_t Sq, int64_t Sk, int64_t heads, int64_t kv_heads, int64_t dh,
               float scale, int causal, const int32_t* q_start, int rows) {
  CNHIP_REQUIRE(B > 0 && Sq > 0 && Sk > 0 && heads > 0 && kv_heads > 0 && dh > 0,
                "%s: bad shape B=%lld Sq=%lld Sk=%lld heads=%lld kv_heads=%lld head_dim=%lld", who, (long long)B,
                (long long)Sq, (long long)Sk, (long long)heads, (long long)kv_heads, (long long)dh);
  CNHIP_REQUIRE(heads % kv_heads == 0, "%s: heads %lld is no multiple of kv_heads %lld", who, (long long)heads,
                (long long)kv_heads);
  if (dh > kMaxHeadDim) {
    set_error("%s: head_dim %lld exceeds %d", who, (long long)dh, kMaxHeadDim);
    return CNHIP_EUNSUPPORTED;
  }
  CNHIP_REQUIRE(rows == CNHIP_ROWS_REF || rows == CNHIP_ROWS_BY_SAMPLE, "%s: bad row order %d", who, rows);
  CNHIP_REQUIRE(causal == 0 || causal == 1, "%s: causal must be 0 or 1", who);
  CNHIP_REQUIRE(causal || !q_start, "%s: q_start needs causal", who);
  CNHIP_REQUIRE(std::isfinite(scale), "%s: scale is not finite", who);
  CNHIP_REQUIRE(B <= 65535 && heads <= 65535 && B * heads <= 65535, "%s: B * heads exceeds 65535", who);
  CNHIP_REQUIRE(Sq < (1 << 30) && Sk < (1 << 30) && Sq * (heads / kv_heads) < (int64_t)1 << 31,
                "%s: sequence too long", who);
  return CNHIP_OK;
}

AttArgs base_args(const float* q, const float* k, const float* v, int64_t B, int64_t Sq, int64_t Sk, int64_t heads,
                  int64_t kv_heads, int64_t dh, float scale, int causal, const int32_t* k_len, const int32_t* q_start,
                  int rows) {
  AttArgs a{};
  a.q = seq(q, B, Sq, rows);
  a.k = seq(k, B, Sk, rows);
  a.v = seq(v, B, Sk, rows);
  a.B = (int)B;
  a.Sq = (int)Sq;
  a.Sk = (int)Sk;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.dh = (int)dh;
  a.group = (int)(heads / kv_heads);
  a.scale = scale;
  a.causal = causal;
  a.k_len = k_len;
  a.q_start = q_start;
  a.lse_sample = rows == CNHIP_ROWS_REF ? 1 : Sq;
  a.lse_row = rows == CNHIP_ROWS_REF ? B : 1;
  a.lse_col = B * Sq;
  return a;
}

}  // namespace
}  // namespace cnhip

using cnhip::as_stream;

extern "C" {

int cnhip_attention_forward(const float* q, const float* k, const float* v, float* out, float* lse, int64_t B,
                            int64_t Sq, int64_t Sk, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale,
                            int causal, const int32_t* k_len, const int32_t* q_start, int rows,
                            cnhip_stream_t stream) {
  const char* who = "cnhip_attention_forward";
  CNHIP_TRY(cnhip::check_args(who, B, Sq, Sk, heads, kv_heads, head_dim, scale, causal, q_start, rows));
  CNHIP_REQUIRE(q && k && v && out, "%s: NULL pointer", who);
  hipStream_t st = as_stream(stream);
  cnhip::AttArgs a =
      cnhip::base_args(q, k, v, B, Sq, Sk, heads, kv_heads, head_dim, scale, causal, k_len, q_start, rows);
  a.out = cnhip::seq(out, B, Sq, rows);
  a.lse = lse;
  const dim3 grid((unsigned)((a.group * Sq + 127) / 128), (unsigned)(B * kv_heads));
  cnhip::dispatch(a.dh, a.k.row == 1, [&](auto d, auto unit) {
    hipLaunchKernelGGL((cnhip::att_fwd_kernel<d(), unit()>), grid, dim3(cnhip::NT), 0, st, a);
  });
  return cnhip::check_launch(who);
}

int cnhip_attention_backward(const float* q, const float* k, const float* v, const float* out, const float* lse,
                             const float* dout, float* dq, float* dk, float* dv, int64_t B, int64_t Sq, int64_t Sk,
                             int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, int causal,
                             const int32_t* k_len, const int32_t* q_start, int rows, cnhip_stream_t stream) {
  const char* who = "cnhip_attention_backward";
  CNHIP_TRY(cnhip::check_args(who, B, Sq, Sk, heads, kv_heads, head_dim, scale, causal, q_start, rows));
  CNHIP_REQUIRE(q && k && v && out && lse && dout && dq && dk && dv, "%s: NULL pointer", who);
  hipStream_t st = as_stream(stream);
  cnhip::AttArgs a =
      cnhip::base_args(q, k, v, B, Sq, Sk, heads, kv_heads, head_dim, scale, causal, k_len, q_start, rows);
  a.o = cnhip::seq(out, B, Sq, rows);
  a.dout = cnhip::seq(dout, B, Sq, rows);
  a.dq = cnhip::seq(dq, B, Sq, rows);
  a.dk = cnhip::seq(dk, B, Sk, rows);
  a.dv = cnhip::seq(dv, B, Sk, rows);
  a.lse_in = lse;
  void* ws = nullptr;
  CNHIP_TRY(cnhip::scratch(st, cnhip::kScratchLayer, (size_t)(B * heads * Sq) * sizeof(float), &ws, who));
  a.delta = static_cast<float*>(ws);
  hipLaunchKernelGGL(cnhip::att_delta_kernel, dim3((unsigned)((Sq + cnhip::NT - 1) / cnhip::NT), (unsigned)(B * heads)),
                     dim3(cnhip::NT), 0, st, a);
  CNHIP_TRY(cnhip::check_launch(who));
  cnhip::dispatch(a.dh, a.k.row == 1, [&](auto d, auto unit) {
    hipLaunchKernelGGL((cnhip::att_dkv_kernel<d(), unit()>),
                       dim3((unsigned)((Sk + 127) / 128), (unsigned)(B * kv_heads)), dim3(cnhip::NT), 0, st, a);
  });
  CNHIP_TRY(cnhip::check_launch(who));
  cnhip::dispatch(a.dh, a.k.row == 1, [&](auto d, auto unit) {
    hipLaunchKernelGGL((cnhip::att_dq_kernel<d(), unit()>),
                       dim3((unsigned)((a.group * Sq + 127) / 128), (unsigned)(B * kv_heads)), dim3(cnhip::NT), 0, st,
                       a);
  });
  return cnhip::check_launch(who);
}

}  // extern "C"
