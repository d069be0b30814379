// Multi-head attention that keeps no probabilities: forward with the row
// log-sum-exp, and the backward that forms the probabilities again from it.
//
//   S = scale q k^T over the keys a query reads,  lse_i = log sum_j exp(S_ij),
//   P_ij = exp(S_ij - lse_i),  out = P v;
//   delta_i = sum_d dout_id out_id,  dS = P (dout v^T - delta) scale,
//   dq = dS k,  dk = dS^T q,  dv = P^T dout   (dk, dv summed over the query
//   heads that share a key head).
//
// Three ways, by rules whose comments measure both sides: single tokens on the
// vector ALUs (att_few_kernel), a forward of few queries on fp32 MFMAs with the
// keys split over blocks (att_fwd_kernel), everything else, the backward above
// all, on the fp16 matrix cores over operands packed as pairs.
//
// On either matrix core a product's accumulators feed the next one without
// leaving the registers.  An accumulator of 32 x 32 holds for its column (lane &
// 31) the rows 8 (r / 4) + 4 (lane / 32) + r % 4, and a B operand holds for its
// column some k's per half-wave, so the order in which the other operand's k's are
// taken can be that of the accumulator.  So the scores are formed with the
// contraction of the product that follows along their rows: S^T = k q^T for out
// and dq (keys along the rows, a query per lane, whose maximum, sum and rescaling
// are the lane's own), S = q k^T for dk and dv (queries along the rows, a key per
// lane).
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "mfma_pair.hpp"

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

// The position of the first query of sample b, and the sample's keys: those past
// its last query's are not among them, so a cache may hold anything there.
__device__ __forceinline__ int64_t start_of(const AttArgs& a, int b) {
  return a.q_start ? (int64_t)a.q_start[b] : (int64_t)a.Sk - a.Sq;
}
__device__ __forceinline__ int keys_of(const AttArgs& a, int b) {
  int64_t n = a.k_len ? min(a.k_len[b], a.Sk) : a.Sk;
  if (a.causal) n = min(n, start_of(a, b) + a.Sq);
  return (int)max(n, (int64_t)0);
}
// Keys that query i reads: the first limit(..) of the sample's n.
__device__ __forceinline__ int limit(const AttArgs& a, int n, int64_t start, int64_t i) {
  if (!a.causal) return n;
  const int64_t l = start + i + 1;
  return (int)(l < 0 ? 0 : l < n ? l : n);
}

constexpr int RT = 32;       // rows of a streamed tile
constexpr int LS = RT + 4;   // floats between features of a tile in LDS
constexpr int NT = 256;      // threads of a block

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

// Forward of few queries.  A block owns 32 rows of a key head's queries (row
// g Sq + i is query i of the g-th of the query heads that share the key head,
// so that the queries of a group fill a wave together) and a run of keys,
// whose tiles its four waves take in turn, each staging its own through its
// own part of LDS: no wave waits for another before the end.  There the four
// join their sums, and where the keys are shared out over several blocks
// att_join_kernel joins theirs.  The features of a row lie a whole column apart in
// memory, so a [feature][row] tile in LDS is staged with float4s along the rows as
// it stands, and serves both as the operand whose lanes are rows (one float per
// lane) and as the one whose lanes are features (four rows per float4).  In v_mfma_
// f32_32x32x2f32 register r of a score tile is the B operand of the k pair {8 (r /
// 4) + r % 4, the same + 4}.  Bound by latency at its sizes: 4 samples, 4 heads, 63
// x 63, head_dim 32: 9 us.
struct SplitArgs {
  int splits, tiles_per_split;  // of 32 keys
  float* o;                     // [split][B kv_heads][row tile][feature][32]
  float2* ml;                   // [split][B kv_heads][row tile][32]: maximum (base 2), sum
};

// A wave's [DHP][RT] tile on its way to LDS.
template <int DHP, bool UNIT>
struct WaveTile {
  static constexpr int U = DHP / 8;  // float4s per lane
  f32x4 v[U];
  __device__ __forceinline__ void load(const float* base, int64_t row, int64_t col, int valid, int dh) {
    const int r = 4 * ((int)threadIdx.x & 7), d0 = ((int)threadIdx.x & 63) >> 3;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = d0 + 8 * u;
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
    const int r = 4 * ((int)threadIdx.x & 7), d0 = ((int)threadIdx.x & 63) >> 3;
#pragma unroll
    for (int u = 0; u < U; ++u) *reinterpret_cast<f32x4*>(lds + (d0 + 8 * u) * LS + r) = v[u];
  }
};

// Between a wave's own LDS writes and reads: no other wave touches its part.
__device__ __forceinline__ void own_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}

template <int DHP, bool UNIT>
__global__ void __launch_bounds__(NT) att_fwd_kernel(AttArgs a, SplitArgs p) {
  __shared__ __align__(16) float lds[4][2][DHP * LS];
  __shared__ float2 stat[4][32];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int64_t rows = (int64_t)a.group * a.Sq;
  const int64_t r = (int64_t)blockIdx.x * 32 + (lane & 31);
  const bool held = r < rows;
  const int head = kh * a.group + (int)(held ? r / a.Sq : 0);
  const int64_t i = held ? r % a.Sq : 0;
  const int n = keys_of(a, b);
  const int lim = held ? limit(a, n, start_of(a, b), i) : 0;
  float q[DHP / 2];
  load_row<DHP>(a.q.at(b, i, (int64_t)head * a.dh), a.q.col, held, a.dh, q);
  int most = lim;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  const int t1 = min((most + RT - 1) / RT, ((int)blockIdx.z + 1) * p.tiles_per_split);
  const float c = a.scale * kLog2e;
  const float* kp = a.k.at(b, 0, (int64_t)kh * a.dh);
  const float* vp = a.v.at(b, 0, (int64_t)kh * a.dh);

  f32x16 o[DHP / 32] = {};
  float m = -INFINITY, l = 0.f;  // of t = scale log2(e) s: maximum and sum of 2^(t - m)
  WaveTile<DHP, UNIT> tk, tv;
  auto load = [&](int t) {
    const int64_t j = (int64_t)t * RT;
    tk.load(kp + j * a.k.row, a.k.row, a.k.col, n - t * RT, a.dh);
    tv.load(vp + j * a.v.row, a.v.row, a.v.col, n - t * RT, a.dh);
  };
  int t = (int)blockIdx.z * p.tiles_per_split + wave;
  if (t < t1) load(t);
  for (; t < t1; t += 4) {
    own_lds();
    tk.store(lds[wave][0]);
    tv.store(lds[wave][1]);
    own_lds();
    if (t + 4 < t1) load(t + 4);
    f32x16 s = dot_rows<DHP>(lds[wave][0], q);
    float most_s = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = t * RT + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
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
    add_rows<DHP>(lds[wave][1], s, o);
  }
  l += other_half(l);
  // the four waves' sums to a common maximum; [feature][row] in the wave's part
  if (lane < 32) stat[wave][lane] = float2{m, l};
  __syncthreads();
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][lane & 31].x);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += stat[w][lane & 31].y * __builtin_amdgcn_exp2f(stat[w][lane & 31].x - base);
  const float f = __builtin_amdgcn_exp2f(m - base);
  float* own = &lds[wave][0][0];
#pragma unroll
  for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      own[(32 * d + 8 * (e / 4) + 4 * (lane >> 5) + e % 4) * 32 + (lane & 31)] = o[d][e] * f;
  __syncthreads();
  const int64_t at = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const float inv = 1.f / total;
  float* out = a.out.at(b, i, (int64_t)head * a.dh);
  for (int d = 2 * wave + (lane >> 5); d < a.dh; d += 8) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x += lds[w][0][d * 32 + (lane & 31)];
    if (p.splits > 1) p.o[(at * a.dh + d) * 32 + (lane & 31)] = x;
    else if (held) out[d * a.out.col] = lim > 0 ? x * inv : 0.f;
  }
  if (wave != 0 || lane >= 32) return;
  if (p.splits > 1) p.ml[at * 32 + lane] = float2{top, total};
  else if (a.lse && held) a.lse[b * a.lse_sample + i * a.lse_row + head * a.lse_col] = lim > 0 ? (top + log2f(total)) * kLn2 : -INFINITY;
}

// x[0 .. N) summed over LANES lanes that are UNIT apart.  Of the N sums each ends
// with N / LANES in x[0 ..): the q-th lane with those from q N / LANES on.
template <int N, int LANES, int UNIT, int SIZE>
__device__ __forceinline__ void sum_scatter(float (&x)[SIZE]) {
  if constexpr (LANES > 1) {
    constexpr int at = LANES / 2 * UNIT;
    const bool up = (int)threadIdx.x & at;
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      const float keep = up ? x[e + N / 2] : x[e], give = up ? x[e] : x[e + N / 2];
      x[e] = keep + __shfl_xor(give, at, 64);
      if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // few in flight, for the registers
    }
    sum_scatter<N / 2, LANES / 2, UNIT>(x);
  }
}

// out of feature d of row r of a key head from its sums, with feature 0 the lse.
__device__ __forceinline__ void put_few(const AttArgs& a, int n, int b, int kh, int r, int d, float x, float top, float total) {
  const int head = kh * a.group + r / a.Sq, i = r % a.Sq;
  const bool reads = limit(a, n, start_of(a, b), i) > 0;
  *a.out.at(b, i, (int64_t)head * a.dh + d) = reads ? x / total : 0.f;
  if (d == 0 && a.lse)
    a.lse[b * a.lse_sample + i * a.lse_row + head * a.lse_col] = reads ? (top + log2f(total)) * kLn2 : -INFINITY;
}

// waves of a SIMD that the registers allow
constexpr int few_waves(int dhp, int r) { return dhp * r > 512 ? 1 : 2; }

// Forward of a key head with up to R query rows (4 or 8), single tokens above
// all: half a flop a byte of the cache and row, which the vector ALUs keep up with,
// where a matrix instruction would fill 32 rows for them.  A wave takes tiles of
// 32 keys as they lie in memory: lane l has keys 4 (l % 8) .. + 3 of features l / 8
// + 8 i, so every load is a float4 and nothing is staged.  The lanes' parts of the
// scores are summed so that each ends with one row's four, whose softmax is its
// part; the probabilities reach the other lanes through LDS, and each lane sums
// its own keys' share of its own features of out until the end.  The loads run a
// chunk of C features ahead.
//
// Bound by the cache's bytes.  16 samples of 4096 keys, head_dim 128 (268 MB),
// with the joining launch: 16 heads on 4 47 us (5.6 TB/s; the kernel of 32 rows
// 94), 32 on 4 72 (95); one sample of 16384, 64 on 8 (134 MB) 50 (126); 64 samples
// of 1024, 8 on 8, head_dim 64 (268 MB) 42 (70).
template <int DHP, int R, bool UNIT>
__global__ void __launch_bounds__(NT, few_waves(DHP, R)) att_few_kernel(AttArgs a, SplitArgs p) {
  constexpr int G = 8, L = 64 / G, TK = 4 * L, NF = DHP / G, C = 4, NC = NF / C, OWN = R * NF / L;
  __shared__ __align__(16) float qs[DHP][R];       // the rows, scaled by nothing
  __shared__ __align__(16) f32x4 ps[4][R][L];     // a wave's probabilities of a row and 4 keys
  __shared__ __align__(16) float fs[4][R];         // and its rows' rescaling
  __shared__ float os[4][R][DHP];
  __shared__ float2 stat[4][R];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, kq = lane % L, fg = lane / L;
  const int row = fg / (G / R);  // whose softmax this lane does
  const int b = (int)blockIdx.x / a.kv_heads, kh = (int)blockIdx.x % a.kv_heads;
  const int rows = a.group * a.Sq;
  for (int e = (int)threadIdx.x; e < DHP * R; e += NT) {
    const int r = e % R, d = e / R;
    qs[d][r] = r < rows && d < a.dh ? *a.q.at(b, r % a.Sq, (int64_t)(kh * a.group + r / a.Sq) * a.dh + d) : 0.f;
  }
  __syncthreads();
  const int n = keys_of(a, b);
  const int lim = row < rows ? limit(a, n, start_of(a, b), row % a.Sq) : 0;
  const int t1 = min((n + TK - 1) / TK, ((int)blockIdx.y + 1) * p.tiles_per_split);
  const float c = a.scale * kLog2e;
  const float* kp = a.k.at(b, 4 * kq, (int64_t)kh * a.dh + fg);
  const float* vp = a.v.at(b, 4 * kq, (int64_t)kh * a.dh + fg);

  f32x4 x[2][C];
  auto load = [&](f32x4 (&to)[C], int part, int t) {  // parts 0 .. NC - 1 of k, then of v
    int64_t key = part < NC ? a.k.row : a.v.row, col = part < NC ? a.k.col : a.v.col;
    asm volatile("" : "+s"(key), "+s"(col));  // no address is carried from tile to tile
    const int i0 = part % NC * C, valid = n - t * TK - 4 * kq;
    const float* at = (part < NC ? kp : vp) + (t * TK * key + G * i0 * col);
    const bool whole = UNIT && (t + 1) * TK <= n;
#pragma unroll
    for (int u = 0; u < C; ++u, at += G * col) {
      // of the padding there are fewer than 32
      const bool in = G * (i0 + u + 1) <= DHP - 31 || fg + G * (i0 + u) < a.dh;
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      if (whole) {
        if (in) y = *reinterpret_cast<const f32x4u*>(at);
      } else if (in) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < valid) y[e] = at[e * key];
      }
      to[u] = y;
    }
  };
  float o[R * NF] = {};  // [row][feature fg + G i]
  float m = -INFINITY, l = 0.f;  // of the row; l of this lane's keys
  int t = (int)blockIdx.y * p.tiles_per_split + wave;
  if (t < t1) load(x[0], 0, t);
  for (; t < t1; t += 4) {
    float s[R * 4] = {};
    f32x4 pr[R];
#pragma unroll
    for (int part = 0; part < 2 * NC; ++part) {
      if (part + 1 < 2 * NC) load(x[(part + 1) & 1], part + 1, t);
      else if (t + 4 < t1) load(x[0], 0, t + 4);
      __builtin_amdgcn_sched_barrier(0);  // one chunk ahead, no more
      const f32x4(&y)[C] = x[part & 1];
      if (part < NC) {
#pragma unroll
        for (int u = 0; u < C; ++u) {
          asm volatile("" ::: "memory");  // q stays in LDS until it is used
          float q[R];
#pragma unroll
          for (int r = 0; r < R; ++r) q[r] = qs[fg + G * (part * C + u)][r];
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * r + e] = fmaf(y[u][e], q[r], s[4 * r + e]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float& z = o[r * NF + (part - NC) * C + u];
#pragma unroll
            for (int e = 0; e < 4; ++e) z = fmaf(y[u][e], pr[r][e], z);
          }
      }
      if (part != NC - 1) continue;
      sum_scatter<4 * R, R, L * (G / R)>(s);  // s[0 .. 4): the row's scores of this lane's keys
      if (R < G) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __shfl_xor(s[e], L, 64);
      }
      float mn = m;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = t * TK + 4 * kq + e < lim ? s[e] * c : -INFINITY;
        mn = fmaxf(mn, s[e]);
      }
#pragma unroll
      for (int w = L / 2; w > 0; w /= 2) mn = fmaxf(mn, __shfl_xor(mn, w, 64));
      const float base = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m - base);
      f32x4 e4;
#pragma unroll
      for (int e = 0; e < 4; ++e) e4[e] = __builtin_amdgcn_exp2f(s[e] - base);
      l = l * f + ((e4[0] + e4[1]) + (e4[2] + e4[3]));
      const bool moved = __ballot(mn != m) != 0;
      m = mn;
      own_lds();
      ps[wave][row][kq] = e4;  // by G / R lanes alike
      if (kq == 0) fs[wave][row] = f;
      own_lds();
#pragma unroll
      for (int r = 0; r < R; ++r) pr[r] = ps[wave][r][kq];
      if (moved) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float fr = fs[wave][r];
#pragma unroll
          for (int i = 0; i < NF; ++i) o[r * NF + i] *= fr;
        }
      }
    }
  }
  sum_scatter<R * NF, L, 1>(o);
#pragma unroll
  for (int w = L / 2; w > 0; w /= 2) l += __shfl_xor(l, w, 64);
#pragma unroll
  for (int e = 0; e < OWN; ++e) {
    const int at = kq * OWN + e;
    os[wave][at / NF][fg + G * (at % NF)] = o[e];
  }
  if (kq == 0) stat[wave][row] = float2{m, l};
  __syncthreads();
  const int64_t heads = gridDim.x, at = (int64_t)blockIdx.y * heads + blockIdx.x;
  for (int e = (int)threadIdx.x; e < rows * a.dh; e += NT) {
    const int r = e / a.dh, d = e % a.dh;
    float top = -INFINITY, total = 0.f, z = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][r].x);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(stat[w][r].x - base);
      total = fmaf(stat[w][r].y, f, total);
      z = fmaf(os[w][r][d], f, z);
    }
    if (p.splits > 1) {
      p.o[at * rows * a.dh + e] = z;
      if (d == 0) p.ml[at * rows + r] = float2{top, total};
    } else {
      put_few(a, n, b, kh, r, d, z, top, total);
    }
  }
}

// Joins the sums of a key head's runs of keys, in their order; a thread per row
// and feature.
__global__ void __launch_bounds__(NT) att_few_join_kernel(AttArgs a, SplitArgs p) {
  const int b = (int)blockIdx.x / a.kv_heads, kh = (int)blockIdx.x % a.kv_heads, rows = a.group * a.Sq;
  const int e = (int)(blockIdx.y * NT + threadIdx.x);
  if (e >= rows * a.dh) return;
  const int r = e / a.dh, d = e % a.dh;
  float top = -INFINITY, total = 0.f, z = 0.f;
  const int64_t heads = gridDim.x;
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float2 ml[8];
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t at = (int64_t)(s0 + u) * heads + blockIdx.x;
      const bool in = s0 + u < p.splits;
      ml[u] = in ? p.ml[at * rows + r] : float2{-INFINITY, 0.f};
      x[u] = in ? p.o[at * rows * a.dh + e] : 0.f;
    }
    float mn = top;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, ml[u].x);
    const float base = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(top - base);
    total *= f;
    z *= f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float fu = __builtin_amdgcn_exp2f(ml[u].x - base);
      total = fmaf(ml[u].y, fu, total);
      z = fmaf(x[u], fu, z);
    }
    top = mn;
  }
  put_few(a, keys_of(a, b), b, kh, r, d, z, top, total);
}

// Joins the sums of a row tile's runs of keys, in their order; 32 features a
// block, a thread per row and four of them.
__global__ void __launch_bounds__(NT) att_join_kernel(AttArgs a, SplitArgs p) {
  const int lane = (int)threadIdx.x & 31, part = (int)threadIdx.x >> 5;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int64_t rows = (int64_t)a.group * a.Sq;
  const int64_t r = (int64_t)blockIdx.x * 32 + lane;
  if (r >= rows) return;
  const int head = kh * a.group + (int)(r / a.Sq);
  const int64_t i = r % a.Sq, step = (int64_t)gridDim.y * gridDim.x, at = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  float top = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.ml[(at + s * step) * 32 + lane].x);
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f, x[4] = {};
  const int d0 = (int)blockIdx.z * 32 + 4 * part;
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.ml[(at + s * step) * 32 + lane];
    const float f = __builtin_amdgcn_exp2f(ml.x - base);
    total += ml.y * f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d0 + e < a.dh) x[e] = fmaf(p.o[((at + s * step) * a.dh + d0 + e) * 32 + lane], f, x[e]);
  }
  const bool reads = limit(a, keys_of(a, b), start_of(a, b), i) > 0;
  const float inv = 1.f / total;
  float* out = a.out.at(b, i, (int64_t)head * a.dh);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d0 + e < a.dh) out[(d0 + e) * a.out.col] = reads ? x[e] * inv : 0.f;
  if (a.lse && part == 0 && blockIdx.z == 0)
    a.lse[b * a.lse_sample + i * a.lse_row + head * a.lse_col] = reads ? (top + log2f(total)) * kLn2 : -INFINITY;
}

__device__ __forceinline__ float lse2_of(const AttArgs& a, int b, int head, int64_t i) {
  const float l = a.lse_in[b * a.lse_sample + i * a.lse_row + head * a.lse_col];
  return l == -INFINITY ? INFINITY : l * kLog2e;  // a row that reads no key: every 2^(t - inf) is 0
}

// ------------------------------------------------------- packed operands
// Long sequences run on the fp16 matrix cores: q, k, v and dout are packed as
// pairs (mfma_pair.hpp), 32 steps x 16 features a fragment, once for each pass,
// and tiles of 32 keys (or queries) go from memory to LDS as they lie.  A tile
// serves as the operand whose lanes are its rows (ds_read_b128) and, turned by
// ds_read_b64_tr_b16, as the one whose lanes are features.  The order in which
// a turned read takes the rows is that of the accumulator registers, so
// probabilities and their gradients are split into their two terms in the
// registers and multiplied without leaving them.
//
// Scales.  Every block of 32 rows of an operand has a power of two of its own,
// from its largest value.  A score takes the two of its operands out again.
// Where blocks are summed, the sum is kept in the scale of the largest block so
// far: a larger one rescales the sum, of a smaller one the other factor, P or dS,
// carries the difference.  Probabilities are at most 1 and enter times 2^14; dS =
// P (dP - delta) of a block of queries is bounded by 2 max ||dout_i|| max ||v_j||,
// i in the block, whose power of two scales it.
struct PackArgs {
  Seq<const float> x[4];  // q, k, v, dout
  char* p[4];             // [head of a sample][block][fragments]
  int* exp[4];            // [head of a sample][block]: a block's exponent,
  float* norm[4];         // its largest row's Euclidean norm
  int blocks[4];
  int first;              // the operand of block z 0 of the packing launch
};

struct PairArgs {
  AttArgs a;
  PackArgs p;
  float *dk_part, *dv_part;  // [B][heads][dh][Sk], where heads share keys
};

// A block's exponent by a vector load: a scalar load under way turns every wait
// for LDS into one for all of it.
template <class T>
__device__ __forceinline__ T exp_at(const T* p, int64_t i) {
  int zero = 0;
  asm("" : "+v"(zero));
  return p[i + zero];
}
// A sum kept with an exponent, before a block of exponent `next` is added: the
// larger of the two becomes the sum's.  Returns by how much the block's is above
// it.
constexpr int kNoExp = 400;  // of a sum that nothing has been added to
template <int N>
__device__ __forceinline__ int meet_exp(f32x16 (&sum)[N], int& exp, int next) {
  next = __builtin_amdgcn_readfirstlane(next);
  if (next < exp) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[d][e] = pr::times_exp2(sum[d][e], next - exp);
    exp = next;
  }
  return next - exp;
}
// The largest row norm of a head.
__device__ __forceinline__ float most_norm(const PackArgs& p, int which, int64_t bh) {
  float n = 0.f;
  for (int i = threadIdx.x & 63; i < p.blocks[which]; i += 64) n = fmaxf(n, p.norm[which][bh * p.blocks[which] + i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n = fmaxf(n, __shfl_xor(n, o, 64));
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(n)));
}

// The head of an operand that a wave works on, and the rows of its sample that
// count, first .. rows - 1: keys that the sample has, queries that read a key.
// Others are zeros, whatever they hold.
struct Operand {
  int which, b, head;
  int64_t bh;  // head of a sample, counted through
  int first, rows;
};
__device__ __forceinline__ Operand operand(const AttArgs& a, int which, int b, int head) {
  const int n = keys_of(a, b);
  if (which == 1 || which == 2) return Operand{which, b, head, (int64_t)b * a.kv_heads + head, 0, n};
  const int64_t before = a.causal ? -start_of(a, b) : 0;  // queries before the first key
  return Operand{which, b, head, (int64_t)b * a.heads + head, (int)(before < 0 ? 0 : min(before, (int64_t)a.Sq)), n > 0 ? a.Sq : 0};
}

// 32 rows of a head in a wave's registers: features 16 s + 8 (lane / 32) .. + 7 of
// row lane % 32 in v[s], zeros where there are none.
template <int KS>
struct RowBlock {
  float v[KS][8];
  __device__ __forceinline__ void load(const AttArgs& a, const Seq<const float>& x, const Operand& o, int blk) {
    const int lane = (int)threadIdx.x & 63, r = blk * 32 + (lane & 31), d0 = 8 * (lane >> 5);
    const bool held = r >= o.first && r < o.rows;
    const float* q = x.at(o.b, held ? r : 0, (int64_t)o.head * a.dh);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] = held && 16 * s + d0 + e < a.dh ? q[(16 * s + d0 + e) * x.col] : 0.f;
  }
  // the exponent of the wave's largest finite value, and the largest row's norm
  __device__ __forceinline__ int exponent(float* norm, int dh) const {
    uint32_t m = 0;
    float n = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t bits = pr::finite_bits(v[s][e]);
        m = max(m, bits);
        n = fmaf(__uint_as_float(bits), __uint_as_float(bits), n);
      }
    n += other_half(n);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
      n = fmaxf(n, __shfl_xor(n, o, 64));
    }
    // squares that leave the range: the bound by the largest value
    if (norm) *norm = n > 1e-30f && n < 1e37f ? sqrtf(n) : __uint_as_float(m) * sqrtf((float)dh);
    return pr::scale_exp((uint32_t)__builtin_amdgcn_readfirstlane((int)m));
  }
  // step s times f in terms, as this lane's fragment
  __device__ __forceinline__ void terms(int s, float f, pr::f16x8 (&x)[2]) const {
    pr::u32x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w0, w1;
      pr::split2(v[s][2 * e] * f, v[s][2 * e + 1] * f, w0, w1);
      hi[e] = w0;
      lo[e] = w1;
    }
    x[0] = __builtin_bit_cast(pr::f16x8, hi);
    x[1] = __builtin_bit_cast(pr::f16x8, lo);
  }
  // delta of the rows, these being dout's
  __device__ __forceinline__ void delta(const AttArgs& a, const Operand& o, int blk) const {
    const int lane = (int)threadIdx.x & 63, r = blk * 32 + (lane & 31);
    RowBlock<KS> out;
    out.load(a, a.o, o, blk);
    float d = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) d = fmaf(v[s][e], out.v[s][e], d);
    d += other_half(d);
    if (r < a.Sq && lane < 32) a.delta[o.bh * a.Sq + r] = d;
  }
};

// A wave packs 32 rows of a head; of dout it also leaves delta.  Bound by memory:
// 32 x 256, 8 heads of 64, forward and backward 40 us for 218 MB (5.4 TB/s).
template <int KS>
__global__ void __launch_bounds__(NT) att_pack_kernel(PairArgs g) {
  const int lane = (int)threadIdx.x & 63, which = (int)blockIdx.z + g.p.first;
  const int head = (int)blockIdx.y % g.a.heads, blk = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
  if (blk >= g.p.blocks[which] || ((which == 1 || which == 2) && head >= g.a.kv_heads)) return;
  const Operand o = operand(g.a, which, (int)blockIdx.y / g.a.heads, head);
  RowBlock<KS> x;
  x.load(g.a, g.p.x[which], o, blk);
  float norm;
  const int e = x.exponent(&norm, g.a.dh);
  const int64_t at = o.bh * g.p.blocks[which] + blk;
  if (lane == 0) {
    g.p.exp[which][at] = e;
    g.p.norm[which][at] = norm;
  }
  char* q = g.p.p[which] + at * KS * (2 * pr::kFrag);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    pr::f16x8 t[2];
    x.terms(s, pr::exp2i(e), t);
    char* to = q + s * (2 * pr::kFrag) + pr::slot(lane, s);
    *reinterpret_cast<pr::f16x8*>(to) = t[0];
    *reinterpret_cast<pr::f16x8*>(to + pr::kFrag) = t[1];
  }
  if (which == 3) x.delta(g.a, o, blk);
}

// This block's head of a sample and 128 rows of it.  The longest go first (a
// head's last rows under a causal mask): `tile` counts from there, over all
// heads of a tile before the next.  Where the heads divide by the eight XCDs,
// to which consecutive blocks go in turn, each takes a run of them, whose keys
// then stay in its L2.
__device__ __forceinline__ void place(int bid, int heads, int& tile, int& bh) {
  if (heads % 8 == 0) {
    const int per = heads / 8, local = bid >> 3;
    tile = local / per;
    bh = (bid & 7) * per + local % per;
  } else {
    tile = bid / heads;
    bh = bid % heads;
  }
}

// Fragments of this lane's own row: packed feature step s, plane q.
template <int KS>
struct RowFrags {
  pr::f16x8 x[KS][2];
  // base: the head's packed rows
  __device__ __forceinline__ void load(const char* base, int row, bool held) {
    const char* p = base + (int64_t)(row >> 5) * KS * (2 * pr::kFrag);
    const int l = ((int)threadIdx.x & 32) | (row & 31);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        x[s][q] = held ? *reinterpret_cast<const pr::f16x8*>(p + (2 * s + q) * pr::kFrag + pr::slot(l, s)) : pr::f16x8{};
  }
};

// acc[x] (rows of a tile x rows of the lanes) = tile[x] row[x]^T over the
// features, for NX pairs of operands at once.  pair(0 .. 7) is called in
// between, for work on the registers of another tile: a MFMA keeps the matrix
// pipe for 32 cycles and the wave for 4, so that work runs beside them.
template <int KS, int NX, class F>
__device__ __forceinline__ void dot_pairs(const char* const (&tile)[NX], const RowFrags<KS>* const (&row)[NX],
                                          f32x16 (&acc)[NX], F&& pair) {
  const int lane = (int)threadIdx.x & 63;
  pr::f16x8 f[2][NX][2];
  auto read = [&](int s) {
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        f[s & 1][x][q] =
            *reinterpret_cast<const pr::f16x8*>(tile[x] + (2 * s + q) * pr::kFrag + pr::slot(lane, s));
  };
  read(0);
#pragma unroll
  for (int x = 0; x < NX; ++x) acc[x] = f32x16{};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    if (s + 1 < KS) read(s + 1);
#pragma unroll
    for (int u = 0; u < 3; ++u)
#pragma unroll
      for (int x = 0; x < NX; ++x)
        acc[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[s & 1][x][u == 0], row[x]->x[s][u == 1], acc[x], 0, 0, 0);
#pragma unroll
    for (int p = 8 * s / KS; p < 8 * (s + 1) / KS; ++p) pair(p);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A score tile's registers as the B operand of two steps of 16 rows, in terms.
struct TileFrags {
  pr::u32x4 w[2][2];
  // registers 2 p and 2 p + 1
  __device__ __forceinline__ void split(int p, float a, float b) {
    uint32_t w0, w1;
    pr::split2(a, b, w0, w1);
    w[p / 4][0][p % 4] = w0;
    w[p / 4][1][p % 4] = w1;
  }
  __device__ __forceinline__ pr::f16x8 at(int t, int q) const { return __builtin_bit_cast(pr::f16x8, w[t][q]); }
};

// Products along a tile's rows: acc[x] (features x rows of the lanes) += tile[x]^T
// p[x], for NX operands at once.  Element i of half-wave h in half t of p is row
// 16 t + 8 (i / 4) + 4 h + i % 4.  The work goes in groups of two blocks of 32
// features (successive MFMAs then do not depend on each other), half 0 of all
// operands before half 1; a group's fragments are read during the one before.
// beside(g) is called in group g, for work on other registers.
template <int KS, int NX>
struct Adder {
  static constexpr int W = KS / 2, G = (W + 1) / 2;  // feature blocks, and groups of two
  static constexpr int GROUPS = 2 * NX * G, HALF = NX * G;
  pr::f16x8 f[2][2][2];

  __device__ __forceinline__ static pr::f16x8 frag(const char* tile, int i, int t, int q) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int lane = (int)threadIdx.x & 63, j = lane & 15, g = lane >> 4 & 1, half = (j & 3) >> 1;
    const int row = 4 * (lane >> 5) + (j >> 2), turn = half * 4 + g * 8;
    const char* at = tile + g * (2 * pr::kFrag) + half * 512 + (j & 1) * 8 + t * 256 + 2 * i * (2 * pr::kFrag) + q * pr::kFrag;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (row ^ turn) * 16));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + ((row + 8) ^ turn) * 16));
    return __builtin_bit_cast(pr::f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ void read(const char* const (&tile)[NX], int g) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (2 * (g % G) + x < W)
#pragma unroll
        for (int q = 0; q < 2; ++q) f[g & 1][x][q] = frag(tile[g / G % NX], 2 * (g % G) + x, g / HALF, q);
  }
  // after read(tile, 0)
  template <class F>
  __device__ __forceinline__ void run(const char* const (&tile)[NX], const TileFrags* const (&p)[NX],
                                      f32x16 (*const (&acc)[NX])[W], F&& beside) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + 1 < GROUPS) read(tile, g + 1);
#pragma unroll
      for (int u = 0; u < 3; ++u)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = 2 * (g % G) + x;
          if (i >= W) continue;
          f32x16& o = (*acc[g / G % NX])[i];
          o = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[g & 1][x][u == 0], p[g / G % NX]->at(g / HALF, u == 1), o, 0, 0, 0);
        }
      beside(g);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};
// calls pair(4 t .. 4 t + 3), the work on a half's registers: part of `parts`
template <class F>
__device__ __forceinline__ void pairs_of(int t, int part, int parts, F&& pair) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e * parts / 4 == part) pair(4 * t + e);
}

// Copies a packed tile into LDS, its fragments shared out among the block's
// four waves.
template <int KS>
__device__ __forceinline__ void copy_tile(const char* tile, char* lds) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < KS / 2; ++u) {
    const int at = (4 * u + wave) * pr::kFrag;
    pr::copy16(tile + at + lane * 16, lds + at);
  }
}

// Tiles that a wave's rows [r0, r0 + 32) reach: their keys' limits grow with
// the row.
__device__ __forceinline__ int tiles_read(const AttArgs& a, int n, int64_t start, int r0) {
  return r0 >= a.Sq ? 0 : (limit(a, n, start, min(r0 + 31, a.Sq - 1)) + 31) / 32;
}

constexpr float kPExp = 14.f;  // probabilities enter times 2^14

// scale log2(e) over the packed operands' scales.  Neither zero, so that times the
// score of a key that is not read it stays infinite, nor infinite, so that times a
// score of zero it stays zero.
__device__ __forceinline__ float score_factor(const AttArgs& a, int exps) {
  const float c = __builtin_amdgcn_fmed3f(pr::times_exp2(fabsf(a.scale) * kLog2e, -exps), 0x1p-126f, 0x1p127f);
  return a.scale < 0.f ? -c : c;  // as unread keys' scores have it, also at a scale of -0
}

// Forward: a wave holds 32 queries of one head and streams the keys and values,
// which a block's four waves share through LDS.  Scores of the next tile are formed
// beside the probabilities of this one.  Bound by the fp16 matrix cores (341
// TFLOP/s of fp32 products at a large library product's rate): 2 x 4096 causal, 16
// heads of 128, 452 us (304 TFLOP/s).
template <int DHP>
__global__ void __launch_bounds__(NT, 2) att_fwd_pair_kernel(PairArgs g, int tiles) {
  constexpr int KS = DHP / 16, TILE = KS * 2 * pr::kFrag;
  __shared__ __align__(16) char kbuf[2][TILE], vbuf[2][TILE];
  const AttArgs& a = g.a;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int tile, bh;
  place((int)blockIdx.x, a.B * a.heads, tile, bh);
  tile = tiles - 1 - tile;
  const int b = bh / a.heads, head = bh % a.heads, kh = head / a.group;
  const int64_t bkh = (int64_t)b * a.kv_heads + kh;
  const int i = tile * 128 + 32 * wave + (lane & 31);
  const bool held = i < a.Sq;
  const int n = keys_of(a, b);
  const int64_t start = start_of(a, b);
  const int lim = held ? limit(a, n, start, i) : 0;
  const int row0 = tile * 128 + 32 * __builtin_amdgcn_readfirstlane(wave);
  const int mine = tiles_read(a, n, start, row0), all = (limit(a, n, start, min(tile * 128 + 127, a.Sq - 1)) + 31) / 32;
  const int *kexp = g.p.exp[1] + bkh * g.p.blocks[1], *vexp = g.p.exp[2] + bkh * g.p.blocks[2];
  RowFrags<KS> q;
  int eq;
  {
    RowBlock<KS> x;
    x.load(a, a.q, operand(a, 0, b, head), row0 / 32);
    eq = x.exponent(nullptr, a.dh);
    const float f = a.scale < 0.f ? -pr::exp2i(eq) : pr::exp2i(eq);  // the scale's sign enters here
#pragma unroll
    for (int u = 0; u < KS; ++u) x.terms(u, f, q.x[u]);
  }
  const char* kp = g.p.p[1] + bkh * g.p.blocks[1] * TILE;
  const char* vp = g.p.p[2] + bkh * g.p.blocks[2] * TILE;
  f32x16 o[DHP / 32] = {};
  float m = -INFINITY, l = 0.f;  // maximum of t = scale log2(e) s, sum of 2^(14 + t - m)
  // Step t forms the scores of tile t, and beside them the probabilities of
  // tile t - 1, which then multiply its values.
  f32x16 s[1] = {};
  TileFrags p;
  float base = 0.f, c = 0.f, part = 0.f;
  int ev = kNoExp;  // the exponent of o
  // tile t's scores masked, the maximum and what it rescales; ek, the exponents
  // of the tile's keys, and dv, by how much that of its values is above ev
  auto top = [&](int t, int ek, int dv) {
    // of no sign: it is in q
    c = fabsf(score_factor(a, eq + ek));
    if (!__all(lim >= 32 * t + 32)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = 32 * t + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        s[0][e] = j < lim ? s[0][e] : -INFINITY;
      }
    }
    float most = s[0][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) most = fmaxf(most, s[0][e]);
    const float mn = fmaxf(m, fmaxf(most, other_half(most)) * c);
    if (__any(mn > m)) {
      const float f = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
      l *= f;
#pragma unroll
      for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= f;
      m = mn;
    }
    base = m == -INFINITY ? 0.f : m;
    if (__any(fabsf(base) >= 0x1p23f)) {
      // The 14 is lost in a maximum of 2^24 and more, and c times a score there is
      // rounded by as much as it: the difference is taken first, of the product as
      // it was rounded for the maximum, so that the largest gives 0.
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = pr::opaque(s[0][e] * c) - base;
      c = 1.f;
      base = 0.f;
    }
    base = base - kPExp + (float)dv;
    part = 0.f;
  };
  auto pair = [&](const f32x16& x, int e) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(x[2 * e], c, -base)), p1 = __builtin_amdgcn_exp2f(fmaf(x[2 * e + 1], c, -base));
    part += p0 + p1;
    p.split(e, p0, p1);
  };
  const RowFrags<KS>* const rows[1] = {&q};
  const TileFrags* const probs[1] = {&p};
  f32x16 (*const sums[1])[KS / 2] = {&o};
  if (all > 0) copy_tile<KS>(kp, kbuf[0]);
  int ek = 0, evt = 0;  // tile t - 1's
  for (int t = 0; t <= all; ++t) {
    pr::wait_and_meet<0>();
    const int u = min(t, all - 1), ek_next = all > 0 ? exp_at(kexp, u) : 0, ev_next = all > 0 ? exp_at(vexp, u) : 0;
    if (t + 1 < all) copy_tile<KS>(kp + (int64_t)(t + 1) * TILE, kbuf[(t + 1) & 1]);
    if (t < all) copy_tile<KS>(vp + (int64_t)t * TILE, vbuf[t & 1]);
    if (t > mine) continue;
    const char* const now[1] = {kbuf[t & 1]};
    if (t == 0) {
      if (mine > 0) dot_pairs<KS, 1>(now, rows, s, [](int) {});
      ek = ek_next;
      evt = ev_next;
      continue;
    }
    // Values below 2^-60 of the largest are multiplied by probabilities that the
    // terms hold as zeros: they add nothing, but for those that are not finite.
    const int dv = min(meet_exp(o, ev, evt), 60);
    top(t - 1, ek, dv);
    ek = ek_next;
    evt = ev_next;
    const char* const before[1] = {vbuf[(t - 1) & 1]};
    Adder<KS, 1> add;
    if (t < mine) {
      f32x16 next[1];
      dot_pairs<KS, 1>(now, rows, next, [&](int e) {
        if (e == 7) add.read(before, 0);
        pair(s[0], e);
      });
      s[0] = next[0];
    } else {
      add.read(before, 0);
      // opaque, or the exponentials of both branches move ahead of them
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = pr::opaque(s[0][e]);
#pragma unroll
      for (int e = 0; e < 8; ++e) pair(s[0], e);
    }
    l += pr::times_exp2(part, dv);
    add.run(before, probs, sums, [](int) {});
  }
  l += other_half(l);
  const float f = 1.f / l;
#pragma unroll
  for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = lim > 0 ? pr::times_exp2(o[d][e] * f, -ev) : 0.f;
  store_row<DHP>(a.out.at(b, held ? i : 0, (int64_t)head * a.dh), a.out.col, held, a.dh, 1.f, o);
  if (a.lse && held && lane < 32)
    a.lse[b * a.lse_sample + i * a.lse_row + head * a.lse_col] =
        lim > 0 ? (m + log2f(pr::times_exp2(l, -(int)kPExp))) * kLn2 : -INFINITY;
}

// A probability times 2^top from its score and its row's lse (base 2) less top.
// The score's and the lse's own errors may take it above 1, by any power of two
// where scores or the products that cancel in them are 2^22 and more: it is held
// to 1, which the scales of P and dS rely on (a NaN stays one).
__device__ __forceinline__ float prob(float s, float c, float lse, float top) {
  return __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(fmaf(s, c, -lse), top));
}

// The exponent of dS of a block of queries: 2 max ||dout|| max ||v|| bounds it.
__device__ __forceinline__ int grad_exp(float dout_norm, float v_norm) {
  return pr::scale_exp(__float_as_uint(fminf(2.f * dout_norm * v_norm, 3e38f)));
}

// LDS of a block of the backward: two tiles of each of two operands.
template <int DHP>
struct GradLds {
  __align__(16) char buf[2][2][DHP / 16 * 2 * pr::kFrag];
  __align__(16) float stat[2][2][32];  // lse (base 2) - 14, scaled delta of the tiles' queries
};

// dq: a wave holds 32 queries of one head and streams keys and values.
template <int DHP>
__device__ __forceinline__ void dq_block(const PairArgs& g, int bid, int tiles, GradLds<DHP>& lds) {
  constexpr int KS = DHP / 16, TILE = KS * 2 * pr::kFrag;
  auto& kbuf = lds.buf[0];
  auto& vbuf = lds.buf[1];
  const AttArgs& a = g.a;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int tile, bh;
  place(bid, a.B * a.heads, tile, bh);
  tile = tiles - 1 - tile;
  const int b = bh / a.heads, head = bh % a.heads, kh = head / a.group;
  const int64_t bkh = (int64_t)b * a.kv_heads + kh;
  const int i = tile * 128 + 32 * wave + (lane & 31);
  const bool held = i < a.Sq;
  const int n = keys_of(a, b);
  const int64_t start = start_of(a, b);
  const int lim = held ? limit(a, n, start, i) : 0;
  const int row0 = tile * 128 + 32 * __builtin_amdgcn_readfirstlane(wave);
  const int mine = tiles_read(a, n, start, row0), all = (limit(a, n, start, min(tile * 128 + 127, a.Sq - 1)) + 31) / 32;
  const int own = min(row0 / 32, g.p.blocks[0] - 1);
  const int ed = grad_exp(g.p.norm[3][(int64_t)bh * g.p.blocks[3] + own], most_norm(g.p, 2, bkh));
  const int eq = g.p.exp[0][(int64_t)bh * g.p.blocks[0] + own], eg = g.p.exp[3][(int64_t)bh * g.p.blocks[3] + own];
  const int *kexp = g.p.exp[1] + bkh * g.p.blocks[1], *vexp = g.p.exp[2] + bkh * g.p.blocks[2];
  const float none = a.scale < 0.f ? INFINITY : -INFINITY;  // the score of a key that is not read
  RowFrags<KS> q, go;
  q.load(g.p.p[0] + (int64_t)bh * g.p.blocks[0] * TILE, held ? i : 0, held);
  go.load(g.p.p[3] + (int64_t)bh * g.p.blocks[3] * TILE, held ? i : 0, held);
  const float lse = held ? lse2_of(a, b, head, i) : INFINITY;
  const float delta0 = held ? pr::times_exp2(a.delta[(int64_t)bh * a.Sq + i], ed) : 0.f;
  float c = 0.f, cd = 0.f, delta = 0.f;
  const char* kp = g.p.p[1] + bkh * g.p.blocks[1] * TILE;
  const char* vp = g.p.p[2] + bkh * g.p.blocks[2] * TILE;
  f32x16 acc[DHP / 32] = {};
  int ek = kNoExp;  // the exponent of acc, less that of dS
  // dS of a tile's first 16 keys is formed, then that of the others beside the
  // product of the first
  f32x16 s[2];
  TileFrags p;
  auto pair = [&](int e) {
    float d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      d[u] = prob(s[0][2 * e + u], c, lse, 0.f) * fmaf(s[1][2 * e + u], cd, -delta);
    p.split(e, d[0], d[1]);
  };
  const RowFrags<KS>* const rows[2] = {&q, &go};
  const TileFrags* const probs[1] = {&p};
  f32x16 (*const sums[1])[KS / 2] = {&acc};
  int ekt = 0, evt = 0;  // the next tile's
  if (all > 0) {
    copy_tile<KS>(kp, kbuf[0]);
    copy_tile<KS>(vp, vbuf[0]);
    ekt = exp_at(kexp, 0);
    evt = exp_at(vexp, 0);
  }
  for (int t = 0; t < all; ++t) {
    pr::wait_and_meet<0>();
    const int over = meet_exp(acc, ek, ekt);
    c = score_factor(a, eq + ekt);
    cd = pr::times_exp2(1.f, ed - eg - evt - over);
    delta = pr::times_exp2(delta0, -over);
    if (t + 1 < all) {
      copy_tile<KS>(kp + (int64_t)(t + 1) * TILE, kbuf[(t + 1) & 1]);
      copy_tile<KS>(vp + (int64_t)(t + 1) * TILE, vbuf[(t + 1) & 1]);
      ekt = exp_at(kexp, t + 1);
      evt = exp_at(vexp, t + 1);
    }
    if (t >= mine) continue;
    const char* const now[2] = {kbuf[t & 1], vbuf[t & 1]};
    dot_pairs<KS, 2>(now, rows, s, [](int) {});
    const char* const keys[1] = {now[0]};
    Adder<KS, 1> add;
    add.read(keys, 0);
    if (!__all(lim >= 32 * t + 32)) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[0][e] = 32 * t + 8 * (e / 4) + 4 * (lane >> 5) + e % 4 < lim ? s[0][e] : none;
    }
    pairs_of(0, 0, 1, pair);
    add.run(keys, probs, sums, [&](int n) { pairs_of(1, n, add.HALF, pair); });
  }
#pragma unroll
  for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = lim > 0 ? pr::times_exp2(acc[d][e], -ek - ed) : 0.f;
  store_row<DHP>(a.dq.at(b, held ? i : 0, (int64_t)head * a.dh), a.dq.col, held, a.dh, a.scale, acc);
}

// dk, dv: a wave holds 32 keys and streams the queries and output gradients of
// one query head; where heads share the keys, into sums of their own
// ([head of a sample][feature][key], att_share_kernel adds them).
template <int DHP>
__device__ __forceinline__ void dkv_block(const PairArgs& g, int bid, GradLds<DHP>& lds) {
  constexpr int KS = DHP / 16, TILE = KS * 2 * pr::kFrag;
  auto& qbuf = lds.buf[0];
  auto& gbuf = lds.buf[1];
  auto& stat = lds.stat;
  const AttArgs& a = g.a;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int tile, bh;
  place(bid, a.B * a.heads, tile, bh);  // the first keys are read by the most queries
  const int b = bh / a.heads, head = bh % a.heads, kh = head / a.group;
  const int64_t bkh = (int64_t)b * a.kv_heads + kh;
  const int key0 = tile * 128, key = key0 + 32 * wave + (lane & 31);
  const int n = keys_of(a, b);
  const int64_t start = start_of(a, b);
  const bool held = key < n;
  const float v_norm = most_norm(g.p, 2, bkh);
  const int own = min(key0 / 32 + __builtin_amdgcn_readfirstlane(wave), g.p.blocks[1] - 1);
  const int ek = g.p.exp[1][bkh * g.p.blocks[1] + own], ev = g.p.exp[2][bkh * g.p.blocks[2] + own];
  const int *qexp = g.p.exp[0] + (int64_t)bh * g.p.blocks[0], *gexp = g.p.exp[3] + (int64_t)bh * g.p.blocks[3];
  const float* gnorm = g.p.norm[3] + (int64_t)bh * g.p.blocks[3];
  const float none = a.scale < 0.f ? INFINITY : -INFINITY;  // the score of a key that is not read
  float c = 0.f, cd = 0.f, top = 0.f;
  RowFrags<KS> k, v;
  k.load(g.p.p[1] + bkh * g.p.blocks[1] * TILE, held ? key : 0, held);
  v.load(g.p.p[2] + bkh * g.p.blocks[2] * TILE, held ? key : 0, held);
  // the first tile of queries that reads the block's first key
  int64_t first = a.causal ? key0 - start : 0;
  first = first < 0 ? 0 : first / 32;
  const int total = key0 < n && first * 32 < a.Sq ? (int)((a.Sq + 31) / 32 - first) : 0;
  const char* qp = g.p.p[0] + ((int64_t)bh * g.p.blocks[0] + first) * TILE;
  const char* gp = g.p.p[3] + ((int64_t)bh * g.p.blocks[3] + first) * TILE;
  f32x16 dk[DHP / 32] = {}, dv[DHP / 32] = {};
  // Of the next tile: its exponents, and a query's lse (lanes 0 .. 31) or delta,
  // as loaded: they are on their way with the copies
  int eqt = 0, egt = 0;
  float raw = 0.f, norm = 0.f;
  int edk = kNoExp, edv = kNoExp;  // the exponents of dk and dv
  auto copy = [&](int t) {
    copy_tile<KS>(qp + (int64_t)t * TILE, qbuf[t & 1]);
    copy_tile<KS>(gp + (int64_t)t * TILE, gbuf[t & 1]);
    eqt = exp_at(qexp, first + t);
    egt = exp_at(gexp, first + t);
    norm = exp_at(gnorm, first + t);
    const int64_t i = min((first + t) * 32 + (lane & 31), (int64_t)a.Sq - 1);
    const float* p = lane < 32 ? a.lse_in + b * a.lse_sample + i * a.lse_row + head * a.lse_col
                               : a.delta + (int64_t)bh * a.Sq + i;
    if (wave == 0) raw = *p;
  };
  // A wave's first tile is that of the first query that reads its first key.
  const int64_t skip = a.causal ? key0 + 32 * __builtin_amdgcn_readfirstlane(wave) - start - first * 32 : 0;
  const int from = (int)(skip < 0 ? 0 : skip / 32 < total ? skip / 32 : total);
  // the probabilities and dS of a tile's first 16 queries are formed, then those
  // of the others beside the products of the first
  f32x16 s[2];
  TileFrags p, ds;
  auto pair = [&](const float (*st)[32], int e) {
    const int r = 8 * (e / 2) + 4 * (lane >> 5) + 2 * (e & 1);
    const float2 lse = *reinterpret_cast<const float2*>(&st[0][r]);
    const float2 delta = *reinterpret_cast<const float2*>(&st[1][r]);
    float w[2] = {prob(s[0][2 * e], c, lse.x, top), prob(s[0][2 * e + 1], c, lse.y, top)};
    float d[2] = {w[0] * fmaf(s[1][2 * e], cd, -delta.x), w[1] * fmaf(s[1][2 * e + 1], cd, -delta.y)};
    p.split(e, w[0], w[1]);
    ds.split(e, d[0], d[1]);
  };
  const RowFrags<KS>* const rows[2] = {&k, &v};
  const TileFrags* const probs[2] = {&p, &ds};
  f32x16 (*const sums[2])[KS / 2] = {&dv, &dk};
  if (total > 0) copy(0);
  for (int t = 0; t < total; ++t) {
    // P carries by how much the exponent of the tile's output gradients is above
    // that of dv (by more than 100: they add nothing that is kept), and dS the same
    // of dk; shift: the exponent of dS over that of P
    const int ed = grad_exp(norm, v_norm);
    const int over = meet_exp(dv, edv, egt), over_k = meet_exp(dk, edk, ed + eqt);
    const int shift = ed - over_k - (int)kPExp + over;
    const bool adds = over <= 100;
    c = score_factor(a, eqt + ek);
    cd = adds ? pr::times_exp2(1.f, shift - egt - ev) : 0.f;
    top = kPExp - (float)over;
    if (wave == 0) {
      const bool in = adds && (first + t) * 32 + (lane & 31) < a.Sq;
      float st = lane < 32 ? INFINITY : 0.f;
      if (in && lane >= 32) st = pr::times_exp2(raw, shift);
      else if (in && raw != -INFINITY) st = raw * kLog2e - kPExp + (float)over;
      stat[t & 1][lane >> 5][lane & 31] = st;
    }
    pr::wait_and_meet<0>();
    if (t + 1 < total) copy(t + 1);
    if (t < from) continue;
    const char* const now[2] = {qbuf[t & 1], gbuf[t & 1]};
    dot_pairs<KS, 2>(now, rows, s, [](int) {});
    const char* const turned[2] = {now[1], now[0]};
    Adder<KS, 2> add;
    add.read(turned, 0);
    const int64_t i0 = start + (first + t) * 32;  // the position of the tile's first query
    if (!(__all(held) && (!a.causal || key0 + 32 * wave + 31 <= i0))) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool reads = held && (!a.causal || key <= i0 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4);
        s[0][e] = reads ? s[0][e] : none;
      }
    }
    const float (*const st_now)[32] = stat[t & 1];
    auto work = [&](int e) { pair(st_now, e); };
    pairs_of(0, 0, 1, work);
    add.run(turned, probs, sums, [&](int n) { pairs_of(1, n, add.HALF, work); });
  }
#pragma unroll
  for (int d = 0; d < DHP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      dk[d][e] = pr::times_exp2(dk[d][e], -edk);
      dv[d][e] = pr::times_exp2(dv[d][e], -edv - (int)kPExp);
    }
  const bool stored = key < a.Sk;
  const int at = stored ? key : 0;
  if (a.group == 1) {
    store_row<DHP>(a.dk.at(b, at, (int64_t)kh * a.dh), a.dk.col, stored, a.dh, a.scale, dk);
    store_row<DHP>(a.dv.at(b, at, (int64_t)kh * a.dh), a.dv.col, stored, a.dh, 1.f, dv);
  } else {
    const int64_t o = (int64_t)bh * a.dh * a.Sk + at;
    store_row<DHP>(g.dk_part + o, a.Sk, stored, a.dh, a.scale, dk);
    store_row<DHP>(g.dv_part + o, a.Sk, stored, a.dh, 1.f, dv);
  }
}

// Seven products, of which the scores and dP are formed for dq and again for dk and
// dv: summing dq over blocks of keys instead would take partial sums or an order
// that changes.  2 x 4096 causal, 16 heads of 128 on 4: 1618 us (297 TFLOP/s).
// Both in one launch, so that the blocks of one fill what those of the other leave
// (head_dim 96 then holds dq to one block on a CU).  Backward, two launches and
// one: 4 samples, 4 heads, 63 x 63, head_dim 32 18 and 13 us, 1 x 8, 1024 x 1024,
// 128 178 and 117, 5 x 6, 1001 x 1001, 80 158 and 117, 8 x 8, 1024 x 1024, 128 312
// and 308; 16 x 8, 2048 x 2048, 96 1377 and 1431.
template <int DHP>
__global__ void __launch_bounds__(NT, DHP <= 64 ? 2 : 1) att_grads_pair_kernel(PairArgs g, int dkv_blocks, int tiles) {
  __shared__ GradLds<DHP> lds;
  if ((int)blockIdx.x < dkv_blocks) dkv_block<DHP>(g, (int)blockIdx.x, lds);
  else dq_block<DHP>(g, (int)blockIdx.x - dkv_blocks, tiles, lds);
}

// dk, dv of a key head: the sums of the heads that share it, in their order; a
// thread per key and four features.  2 x 4096, 16 heads of 128 on 4: 168 MB, 50 us.
__global__ void __launch_bounds__(NT) att_share_kernel(PairArgs g) {
  const AttArgs& a = g.a;
  const int key = (int)blockIdx.x * NT + (int)threadIdx.x, widths = (a.dh + 3) / 4;
  if (key >= a.Sk) return;
  const int b = (int)blockIdx.y / a.kv_heads, kh = (int)blockIdx.y % a.kv_heads;
  const int d0 = (int)blockIdx.z % widths * 4;
  const bool v = (int)blockIdx.z >= widths;
  const int64_t head = (int64_t)a.dh * a.Sk;
  const float* part = (v ? g.dv_part : g.dk_part) + ((int64_t)b * a.heads + (int64_t)kh * a.group) * head + key;
  const Seq<float>& out = v ? a.dv : a.dk;
  float* o = out.at(b, key, (int64_t)kh * a.dh);
  float s[4] = {};
#pragma unroll 2
  for (int h = 0; h < a.group; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d0 + e < a.dh) s[e] += part[h * head + (int64_t)(d0 + e) * a.Sk];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d0 + e < a.dh) o[(d0 + e) * out.col] = s[e];
}

// f(the features of a row padded to the kernel's as an integral constant)
template <class F>
void by_width(int dh, F&& f) {
  if (dh <= 32) f(std::integral_constant<int, 32>{});
  else if (dh <= 64) f(std::integral_constant<int, 64>{});
  else if (dh <= 96) f(std::integral_constant<int, 96>{});
  else f(std::integral_constant<int, 128>{});
}

// Lays out the workspace of the packed operands and packs them: k and v, and
// for the backward q and dout too, with whose packing comes delta.
int pack(PairArgs& g, bool backward, hipStream_t st, const char* who) {
  AttArgs& a = g.a;
  PackArgs& p = g.p;
  const int steps = a.dh <= 32 ? 2 : a.dh <= 64 ? 4 : a.dh <= 96 ? 6 : 8;
  p.first = backward ? 0 : 1;
  const int last = backward ? 3 : 2;
  size_t bytes = 0, data[4], exps[4], norms[4];
  auto place_bytes = [&](size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  int most = 0;
  for (int w = p.first; w <= last; ++w) {
    const bool kv = w == 1 || w == 2;
    p.blocks[w] = (int)(((kv ? a.Sk : a.Sq) + 31) / 32);
    most = p.blocks[w] > most ? p.blocks[w] : most;
    const size_t n = (size_t)a.B * (kv ? a.kv_heads : a.heads) * p.blocks[w];
    data[w] = place_bytes(n * steps * 2 * pr::kFrag);
    exps[w] = place_bytes(n * sizeof(int));
    norms[w] = place_bytes(n * sizeof(float));
  }
  const size_t delta = place_bytes(backward ? (size_t)a.B * a.heads * a.Sq * sizeof(float) : 0);
  const size_t sums = backward && a.group > 1 ? (size_t)a.B * a.heads * a.dh * a.Sk * sizeof(float) : 0;
  const size_t dk_part = place_bytes(sums), dv_part = place_bytes(sums);
  void* ws = nullptr;
  CNHIP_TRY(scratch(st, kScratchLayer, bytes, &ws, who));
  char* base = static_cast<char*>(ws);
  g.dk_part = reinterpret_cast<float*>(base + dk_part);
  g.dv_part = reinterpret_cast<float*>(base + dv_part);
  for (int w = p.first; w <= last; ++w) {
    p.p[w] = base + data[w];
    p.exp[w] = reinterpret_cast<int*>(base + exps[w]);
    p.norm[w] = reinterpret_cast<float*>(base + norms[w]);
  }
  a.delta = reinterpret_cast<float*>(base + delta);
  p.x[0] = a.q;
  p.x[1] = a.k;
  p.x[2] = a.v;
  p.x[3] = a.dout;
  by_width(a.dh, [&](auto d) {
    hipLaunchKernelGGL(att_pack_kernel<d() / 16>,
                       dim3((unsigned)((most + 3) / 4), (unsigned)(a.B * a.heads), (unsigned)(last - p.first + 1)), dim3(NT),
                       0, st, g);
  });
  return check_launch(who);
}

// Whether the forward runs on packed operands.  The kernel of few queries splits
// the keys over blocks too, and wins where the queries alone are too few blocks of
// 128: 4 samples, 4 heads, 128 x 128, head_dim 32 7 us against 13 on packed
// operands, 8 x 8, 64 x 1024, 64 36 (56); 32 x 8, 128 x 128, 64 37 (31), 8 x 8, 1024
// x 63, 64 109 (21).
bool pairs_forward(const AttArgs& a) { return a.Sq >= 64 && (int64_t)a.B * a.heads * a.Sq >= 8192; }

constexpr int kMaxHeadDim = 128;
constexpr int64_t kFewRows = 8;  // query rows of a key head that att_few_kernel takes, whose comment measures both sides

template <class T>
Seq<T> seq(T* p, int64_t B, int64_t S, int rows) {
  return rows == CNHIP_ROWS_REF ? Seq<T>{p, 1, B, B * S} : Seq<T>{p, S, 1, B * S};
}

// by_width, and whether a step's neighbours are adjacent
template <class F>
void dispatch(int dh, bool unit, F&& f) {
  by_width(dh, [&](auto d) {
    if (unit) f(d, std::true_type{});
    else f(d, std::false_type{});
  });
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
  CNHIP_REQUIRE(B * heads * (Sq / 128 + Sk / 128 + 2) < (int64_t)1 << 31, "%s: too many rows", who);
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
  if (cnhip::pairs_forward(a)) {
    cnhip::PairArgs g{a, {}, nullptr, nullptr};
    CNHIP_TRY(cnhip::pack(g, false, st, who));
    const int tiles = (int)((Sq + 127) / 128);
    cnhip::by_width(a.dh, [&](auto d) {
      hipLaunchKernelGGL((cnhip::att_fwd_pair_kernel<d()>), dim3((unsigned)(tiles * B * heads)), dim3(cnhip::NT), 0, st,
                         g, tiles);
    });
    return cnhip::check_launch(who);
  }
  if (a.group * Sq <= cnhip::kFewRows) {
    const int R = a.group * Sq <= 4 ? 4 : 8, rows = (int)(a.group * Sq);
    const int64_t tiles = (Sk + 31) / 32;
    // Runs of keys: as many blocks as the CUs hold, at least one tile a wave.
    const int width = (int)((head_dim + 31) / 32 * 32);
    int64_t splits = 256 * cnhip::few_waves(width, R) / (B * kv_heads);
    if (splits > tiles / 4) splits = tiles / 4;
    if (splits < 1) splits = 1;
    cnhip::SplitArgs p{};
    p.tiles_per_split = (int)((tiles + splits - 1) / splits);
    p.splits = (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
    if (p.splits > 1) {
      const size_t all = (size_t)(p.splits * B * kv_heads * rows);
      void* ws = nullptr;
      CNHIP_TRY(cnhip::scratch(st, cnhip::kScratchLayer, all * (sizeof(float2) + head_dim * sizeof(float)), &ws, who));
      p.ml = static_cast<float2*>(ws);
      p.o = reinterpret_cast<float*>(p.ml + all);
    }
    const dim3 grid((unsigned)(B * kv_heads), (unsigned)p.splits);
    cnhip::dispatch(a.dh, a.k.row == 1, [&](auto d, auto unit) {
      if (R == 4) hipLaunchKernelGGL((cnhip::att_few_kernel<d(), 4, unit()>), grid, dim3(cnhip::NT), 0, st, a, p);
      else hipLaunchKernelGGL((cnhip::att_few_kernel<d(), 8, unit()>), grid, dim3(cnhip::NT), 0, st, a, p);
    });
    CNHIP_TRY(cnhip::check_launch(who));
    if (p.splits == 1) return CNHIP_OK;
    hipLaunchKernelGGL(cnhip::att_few_join_kernel,
                       dim3((unsigned)(B * kv_heads), (unsigned)((rows * head_dim + cnhip::NT - 1) / cnhip::NT)),
                       dim3(cnhip::NT), 0, st, a, p);
    return cnhip::check_launch(who);
  }
  // Runs of keys: enough blocks for two on every CU, at least two tiles a wave.
  const int64_t row_tiles = (a.group * Sq + 31) / 32, key_tiles = (Sk + 31) / 32;
  int64_t splits = 512 / (row_tiles * B * kv_heads);
  if (splits > key_tiles / 8) splits = key_tiles / 8;
  if (splits < 1) splits = 1;
  cnhip::SplitArgs p{};
  p.tiles_per_split = (int)((key_tiles + splits - 1) / splits);
  p.splits = (int)((key_tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  CNHIP_REQUIRE(row_tiles < (int64_t)1 << 31, "%s: too many rows", who);
  if (p.splits > 1) {
    const size_t rows32 = (size_t)(p.splits * B * kv_heads * row_tiles) * 32;
    void* ws = nullptr;
    CNHIP_TRY(cnhip::scratch(st, cnhip::kScratchLayer, rows32 * (sizeof(float2) + head_dim * sizeof(float)), &ws, who));
    p.ml = static_cast<float2*>(ws);
    p.o = reinterpret_cast<float*>(p.ml + rows32);
  }
  const dim3 grid((unsigned)row_tiles, (unsigned)(B * kv_heads), (unsigned)p.splits);
  cnhip::dispatch(a.dh, a.k.row == 1, [&](auto d, auto unit) {
    hipLaunchKernelGGL((cnhip::att_fwd_kernel<d(), unit()>), grid, dim3(cnhip::NT), 0, st, a, p);
  });
  CNHIP_TRY(cnhip::check_launch(who));
  if (p.splits == 1) return CNHIP_OK;
  hipLaunchKernelGGL(cnhip::att_join_kernel, dim3((unsigned)row_tiles, (unsigned)(B * kv_heads), (unsigned)((head_dim + 31) / 32)),
                     dim3(cnhip::NT), 0, st, a, p);
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
  cnhip::PairArgs g{a, {}, nullptr, nullptr};
  CNHIP_TRY(cnhip::pack(g, true, st, who));
  const int tiles = (int)((Sq + 127) / 128);
  const unsigned dkv_blocks = (unsigned)((Sk + 127) / 128 * B * heads), dq_blocks = (unsigned)(tiles * B * heads);
  cnhip::by_width(a.dh, [&](auto d) {
    hipLaunchKernelGGL((cnhip::att_grads_pair_kernel<d()>), dim3(dkv_blocks + dq_blocks), dim3(cnhip::NT), 0, st, g,
                       (int)dkv_blocks, tiles);
  });
  CNHIP_TRY(cnhip::check_launch(who));
  if (a.group == 1) return CNHIP_OK;
  hipLaunchKernelGGL(cnhip::att_share_kernel,
                     dim3((unsigned)((Sk + cnhip::NT - 1) / cnhip::NT), (unsigned)(B * kv_heads), (unsigned)((head_dim + 3) / 4 * 2)),
                     dim3(cnhip::NT), 0, st, g);
  return cnhip::check_launch(who);
}

}  // extern "C"
