// fp32 products on the fp16 matrix cores from operands packed as pairs.
//
// An fp32 value times a power of two that puts its operand's largest at 2^15
// is the sum of two fp16 terms, x = x0 + x1 with x0 = fp16(x) and
// x1 = fp16(x - x0), to within 2^-22 of itself (each rounding is to 2^-11; the
// root of the mean square is 2^-24), or to within 2^-39 of the operand's
// largest where that is more: x1 lies on fp16's subnormal grid of 2^-24 once x
// is small.  The matrix cores keep subnormal inputs and products exactly
// (measured: 2^-24 * 2^-24).  A product takes three MFMAs,
//   a1 b0 + a0 b1 + a0 b0,
// into one fp32 accumulator; the term left out is below 2^-22 of a b, as the
// errors of the terms are.  A sum of such products is off by what an fp32 sum
// is (1021 rows of 513: log-sum-exp 4.9e-8 in both, 8192 x 1024 x 32000 gradient
// 5.4e-7 against 3.2e-6 of a library's fp32 product), at a third of the fp16
// rate: half the MFMAs of the split in three bf16 terms (mfma_split.hpp),
// whose wider range the scale replaces.
//
// The matrix core cuts the low bits of a sum towards minus infinity, so long
// sums drift.  A contraction therefore enters its second half with A negated
// and its accumulators with it, and the drifts of the two halves cancel.
//
// Packed layout.  An operand of `rows` rows and a contraction of k is held in
// fragments of 32 rows x 16 k, two planes (x0, x1) of 1024 bytes each: row r's
// eight k of half h (8 h .. 8 h + 7), which lane 32 h + r of the MFMA takes, lie
// in 16 bytes at slot(32 h + r, step).  Fragments of a row block follow each
// other along k.  Both sizes are padded with zeros to multiples of 32.  Such an
// operand goes from memory to LDS as it lies (16 bytes a lane, no registers)
// and from LDS to the MFMA with one ds_read_b128 over the 1024 bytes of a
// plane.  The same packing also serves the product whose contraction runs along
// its rows: ds_read_b64_tr_b16 turns 4 x 16 halves on the way to the registers.
// Half a wave then takes 4 rows of both halves of two steps; slot's permutation
// of the rows spreads those over all 64 banks (unpermuted they met in a
// quarter of them: 6.8 cycles a read for 2).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace cnhip {
namespace pr {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kFrag = 1024;  // bytes of a fragment's plane

// ------------------------------------------------------------------ scales
// A scale is kept as the largest finite |x| of the operand (its bits, so that
// an unsigned maximum orders them).  The operand's exponent is that of the
// power of two which takes it to [2^14, 2^15); at most 126, so that the power
// and its inverse are normal (an operand below 2^-112 stays below 2^14).
__device__ __forceinline__ int scale_exp(uint32_t largest_bits) {
  return min(126, 14 + 127 - (int)(largest_bits >> 23));
}
// 2^e for an operand's exponent
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// x 2^e for any e
__device__ __forceinline__ float times_exp2(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// Byte of lane l's 16 in a plane of step s.
__device__ __forceinline__ int slot(int l, int s) {
  return ((l & 32) | ((l & 31) ^ ((l >> 5) * 4 + (s & 1) * 8))) * 16;
}

// Keeps the compiler from folding the operation that formed x into what uses it.
__device__ __forceinline__ float opaque(float x) {
  asm("" : "+v"(x));
  return x;
}
// Two values to their terms: w0 = {x0(a), x0(b)}, w1 the remainders'.  Values
// and remainders are opaque: a product that is converted at once, or a
// remainder, became a v_fma_mixlo_f16 otherwise, and dq came out ten times less
// exact.
__device__ __forceinline__ void split2(float a, float b, uint32_t& w0, uint32_t& w1) {
  a = opaque(a);
  b = opaque(b);
  const f16x2 h = __builtin_convertvector(f32x2{a, b}, f16x2);
  const f16x2 l = __builtin_convertvector(f32x2{opaque(a - (float)h[0]), opaque(b - (float)h[1])}, f16x2);
  w0 = __builtin_bit_cast(uint32_t, h);
  w1 = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  return m;
}

// This lane's eight k of fragment (block, step) of an operand of `steps` steps.
__device__ __forceinline__ void put_frag(char* p, int64_t block, int steps, int step, const float (&x)[8]) {
  u32x4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t h, l;
    split2(x[2 * e], x[2 * e + 1], h, l);
    hi[e] = h;
    lo[e] = l;
  }
  char* q = p + (block * steps + step) * (2 * kFrag) + slot(threadIdx.x & 63, step);
  *reinterpret_cast<u32x4*>(q) = hi;
  *reinterpret_cast<u32x4*>(q + kFrag) = lo;
}

// ----------------------------------------------------------- global -> LDS
// 16 bytes a lane from `src` (the lane's own address) to lds + 16 lane; lds is
// wave-uniform.  Counted by vmcnt.  Written out because the compiler, where it
// sees such a copy, waits for all of them before every LDS read that turns its
// data; it has no output register, and wait_and_meet orders it.
__device__ __forceinline__ void copy16(const void* src, const char* lds) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds);
  uint32_t m0;  // the register that holds the LDS address is the compiler's: put back
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
      : "=&s"(m0)
      : "s"(at), "v"(src)
      : "memory");
}

// Waits until at most VM of this wave's copies and none of its LDS reads are
// under way, then for the block's other waves.
template <int VM>
__device__ __forceinline__ void wait_and_meet() {
  static_assert(VM < 16, "the count's low four bits");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | VM);  // vmcnt(VM) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// ------------------------------------------------------------------- GEMM
struct Packed {
  const char* p;
  int blocks;  // of 32 rows
  int steps;   // of 16 k
};

struct GemmArgs {
  Packed a, b;
  int M, N;              // output rows (of A) and columns (of B)
  int steps;             // contraction, in steps of 16
  int steps_per_split;   // even
  int half;              // the step where the second half begins
};

// A block of 2 x WN waves, each with 32 MI x 64 of the product, takes a tile of 64 MI x 64
// WN.  WN = 4: one block to a CU, with four LDS buffers for the steps; WN = 2: two, with
// three each, of which one computes while the other stores its tile.  G = 2, for products
// of few tiles: two such groups of waves, four buffers each, share the steps of a tile of
// 128 x 128, so that a SIMD still has two waves, and exchange their sums in LDS: each
// ends with one of the two blocks of 32 columns.
template <int WN_, int MI_ = 4, int G_ = 1>
struct Tile {
  static constexpr int WN = WN_, MI = MI_, G = G_, TM = 64 * MI, TN = 64 * WN, NT = 128 * WN * G;
  static constexpr int J = 2 / G;                    // blocks of 32 columns that a wave ends with
  static constexpr int A = 4 * MI, B = 4 * WN;       // pieces of 1024 bytes a step
  static constexpr int kStage = (A + B) * kFrag;
  static constexpr int kStages = WN == 4 || G == 2 ? 4 : 3;
  static constexpr int kLds = G * kStages * kStage;
  static constexpr int kCopies = (A + B) / (2 * WN);  // a wave's of a step
  static_assert(G == 2 ? WN == 2 && MI == 2 : MI == 4 && (WN == 2 || WN == 4), "tiles");
  static __device__ __forceinline__ int wave() {
    const int w = threadIdx.x >> 6;
    return G == 1 ? w : w % (2 * WN);
  }
  static __device__ __forceinline__ int group() { return G == 1 ? 0 : (int)(threadIdx.x >> 6) / (2 * WN); }
  // the wave's first row and, of its block j, this lane's column in the tile
  static __device__ __forceinline__ int row0() { return wave() / WN * (32 * MI); }
  static __device__ __forceinline__ int column(int j) { return wave() % WN * 64 + 32 * (j + group()) + (int)(threadIdx.x & 31); }
};
constexpr int TM = Tile<4>::TM, TN = Tile<4>::TN, GNT = Tile<4>::NT, kGemmLds = Tile<4>::kLds;

// Staging of one operand: PIECES pieces of 1024 bytes a step, PER a wave.
//   TR false: piece j = plane j & 1 of the fragment of row block j / 2
//   TR true (contraction along the packed rows): piece j = for the 16 output
//     rows of packed step j, both planes of the 16 packed rows of this step:
//     [plane][k half of 8][slot of the row][8 halves]
template <bool TR, int PIECES, int PER>
struct Stage {
  const char* src[PER];
  int64_t step;  // bytes per step (TR: per two steps)
  int lds[PER];
  __device__ __forceinline__ void init(const Packed& o, int tile, int wave) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int j = PER * wave + u;
      lds[u] = j * kFrag;
      if (TR) {
        const int s = min(tile * PIECES + j, o.steps - 1);
        src[u] = o.p + (int64_t)s * (2 * kFrag) + (lane >> 5) * kFrag + ((lane >> 4 & 1) * 32 + (lane & 15)) * 16;
        step = (int64_t)o.steps * (2 * kFrag);
      } else {
        const int b = min(tile * (PIECES / 2) + (j >> 1), o.blocks - 1);
        src[u] = o.p + (int64_t)b * o.steps * (2 * kFrag) + (j & 1) * kFrag + lane * 16;
        step = 2 * kFrag;
      }
    }
  }
  __device__ __forceinline__ void copy(int t, int u, char* buf) const {
    const int64_t at = TR ? (int64_t)(t >> 1) * step + (t & 1) * 256 : (int64_t)t * step;
    copy16(src[u] + at, buf + lds[u]);
  }
};

// This lane's fragment of row block `blk` of the tile, plane q; t: the step.
template <bool TR>
__device__ __forceinline__ f16x8 frag(const char* buf, int blk, int q, int t) {
  const int lane = threadIdx.x & 63;
  if constexpr (!TR) return *reinterpret_cast<const f16x8*>(buf + (2 * blk + q) * kFrag + slot(lane, t));
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int j = lane & 15, g = lane >> 4 & 1, half = (j & 3) >> 1, k = 8 * (lane >> 5) + (j >> 2);
  const char* p = buf + (2 * blk + g) * kFrag + q * 512 + half * 256 + (j & 1) * 8;
  s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (k ^ (half * 4 + g * 8)) * 16));
  s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + ((k + 4) ^ (half * 4 + g * 8)) * 16));
  return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ f16x8 flip(f16x8 x, uint32_t sign) {
  u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] ^= sign;
  return __builtin_bit_cast(f16x8, w);
}

// What a wave holds: MI x 2 accumulators, block (i, j) rows 32 i .. of its 32 MI
// (row 8 (e / 4) + 4 (lane / 32) + e % 4 in element e), columns 32 j + lane % 32
// of its 64.
template <int MI>
struct AccOf {
  f32x16 x[MI][2];
};
using Acc = AccOf<4>;
template <int MI>
struct Frags {
  f16x8 a[MI][2], b[2][2];
};

// Block -> tile.  Consecutive blocks go to the 8 XCDs in turn; each XCD takes
// a contiguous run of tiles, walked in groups of 4 tile rows, so the operands
// of the tiles that run on it at a time fit its L2.
__device__ __forceinline__ void tile_of(int bid, int nm, int nn, int& tm, int& tn) {
  const int total = nm * nn, xcd = bid & 7, local = bid >> 3, base = total >> 3, rem = total & 7;
  const int tile = xcd * base + min(xcd, rem) + local;
  constexpr int G = 4;
  const int per = G * nn, grp = tile / per, first = grp * G, size = min(nm - first, G), in = tile - grp * per;
  tm = first + in % size;
  tn = in / size;
}

// The contraction [t0, t1) of a tile; the sums' sign is right, and with two groups a
// wave's are in x[.][0].  The steps go
// through four LDS buffers (three), three (two) on their way while one is read;
// the fragments of the next step are read while this one's MFMAs run.
template <bool TA, bool TB, class T = Tile<4>>
__device__ __forceinline__ void gemm_tile(const GemmArgs& g, int tm, int tn, int t0, int t1, char* lds,
                                          AccOf<T::MI>& acc) {
  constexpr int kStage = T::kStage, kStages = T::kStages, kCopies = T::kCopies, kBehind = T::A * kFrag;
  constexpr int MI = T::MI, kOfA = T::A / (2 * T::WN), kTurns = 3 * MI, kReads = 2 * MI + 4, kSlots = kTurns / kCopies;
  const int wave = T::wave(), wm = wave / T::WN, wn = wave % T::WN;
  // two groups: the steps of the first, which are as many as the second's or two more
  const int shared = T::G == 1 ? 0 : ((t1 - t0) / 2 + 1) / 2 * 2;
  char* const box = lds;
  if (T::G == 2) {
    lds += __builtin_amdgcn_readfirstlane(T::group()) * (T::kStages * T::kStage);
    if (__builtin_amdgcn_readfirstlane(T::group())) t0 += shared;
    else t1 = t0 + shared;
  }
  Stage<TA, T::A, kOfA> sa;
  Stage<TB, T::B, kCopies - kOfA> sb;
  auto buffer = [&](int t) { return lds + (kStages == 4 ? t & 3 : (int)((unsigned)t % 3u)) * kStage; };
  sa.init(g.a, tm, wave);
  sb.init(g.b, tn, wave);
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc.x[i][j] = f32x16{};
  // piece u (0 .. kCopies - 1) of step t's copies; past the last step the last is
  // copied again, so that the wait counts stay the same
  auto copy = [&](int t, int u) {
    char* buf = buffer(t);
    const int s = t < t1 ? t : t1 - 1;
    if (u < kOfA) sa.copy(s, u, buf);
    else sb.copy(s, u - kOfA, buf + kBehind);
  };
  // fragment u (0 .. kReads - 1) of step t, in the order of their first use
  auto read = [&](int t, int odd, int u, Frags<MI>& f) {
    const char* buf = buffer(t);
    if (u < 2) f.b[u][0] = frag<TB>(buf + kBehind, 2 * wn + u, 0, odd);
    else if (u < MI + 2) f.a[u - 2][1] = frag<TA>(buf, MI * wm + u - 2, 1, odd);
    else if (u < MI + 4) f.b[u - MI - 2][1] = frag<TB>(buf + kBehind, 2 * wn + u - MI - 2, 1, odd);
    else f.a[u - MI - 4][0] = frag<TA>(buf, MI * wm + u - MI - 4, 0, odd);
  };
  Frags<MI> f0, f1;
  auto step = [&](int t, int odd, Frags<MI>& now, Frags<MI>& next) {
    // step t + 1 has arrived (the younger ones may be on their way), and every
    // wave holds step t in registers: its buffer is free
    wait_and_meet<(kStages - 2) * kCopies>();
    if (t == g.half) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc.x[i][j] = -acc.x[i][j];
    }
    const uint32_t sign = t >= g.half ? 0x80008000u : 0u;
    // a MFMA keeps the matrix pipe for 32 cycles and the wave for 4: the reads,
    // copies and sign changes go between them
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int i = u % MI, x = u < MI ? 1 : 0, y = u >= MI && u < 2 * MI ? 1 : 0;
      if (u < 2 * MI) now.a[i][x] = flip(now.a[i][x], sign);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc.x[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now.a[i][x], now.b[j][y], acc.x[i][j], 0, 0, 0);
      constexpr int kTwo = kReads - kTurns;  // turns that read two
      read(t + 1, 1 - odd, u < kTwo ? 2 * u : u + kTwo, next);
      if (u < kTwo) read(t + 1, 1 - odd, 2 * u + 1, next);
      if (u % kSlots == 0 && u / kSlots < kCopies) copy(t + kStages, u / kSlots);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int t = 0; t < kStages; ++t)
#pragma unroll
    for (int u = 0; u < kCopies; ++u) copy(t0 + t, u);
  wait_and_meet<(kStages - 1) * kCopies>();
#pragma unroll
  for (int u = 0; u < kReads; ++u) read(t0, 0, u, f0);
  // t0 is even, so a step's parity, and with it the slots, is known here
  for (int t = t0; t < t1; t += 2) {
    step(t, 0, f0, f1);
    if (t + 1 < t1) step(t + 1, 1, f1, f0);
  }
  if (T::G == 2) {  // both groups meet equally often
    for (int t = t1 - t0; t < shared; ++t) wait_and_meet<0>();
  }
  wait_and_meet<0>();  // the copies that went past the end
  if (t1 > g.half) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc.x[i][j] = -acc.x[i][j];
  }
  if constexpr (T::G == 2) {
    const int lane = threadIdx.x & 63, from = __builtin_amdgcn_readfirstlane(T::group());
    f32x4* to = reinterpret_cast<f32x4*>(box) + (threadIdx.x >> 6) * (4 * MI * 64) + lane;
    const f32x4* other = reinterpret_cast<const f32x4*>(box) + ((threadIdx.x >> 6) ^ 4) * (4 * MI * 64) + lane;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const f32x16 give = from ? acc.x[i][0] : acc.x[i][1];
      if (from) acc.x[i][0] = acc.x[i][1];
#pragma unroll
      for (int q = 0; q < 4; ++q) to[(4 * i + q) * 64] = f32x4{give[4 * q], give[4 * q + 1], give[4 * q + 2], give[4 * q + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = other[(4 * i + q) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc.x[i][0][4 * q + e] += v[e];
      }
  }
}

// p[n + ld m] = value(element), or += for ADD, for the elements of a tile that
// this lane holds and that exist.  ADD reads all of a column before it writes
// one, so the reads are under way together.
template <bool ADD, class T = Tile<4>, class F>
__device__ __forceinline__ void put_tile(const AccOf<T::MI>& acc, int tm, int tn, int M, int N, float* __restrict__ p,
                                         int64_t ld, F&& value) {
  const int lane = threadIdx.x & 63;
  const int m0 = tm * T::TM + T::row0(), m1 = m0 + 4 * (lane >> 5);
#pragma unroll
  for (int j = 0; j < T::J; ++j) {
    const int n = tn * T::TN + T::column(j);
    if (n >= N) continue;
    float* q = p + n + ld * m1;
    auto row = [](int i, int e) { return 32 * i + 8 * (e / 4) + e % 4; };
    if (m0 + 32 * T::MI <= M) {
      float old[T::MI][16];
      if (ADD) {
#pragma unroll
        for (int i = 0; i < T::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) old[i][e] = q[ld * row(i, e)];
      }
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) q[ld * row(i, e)] = ADD ? old[i][e] + value(acc.x[i][j][e]) : value(acc.x[i][j][e]);
    } else {
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (m1 + row(i, e) < M) {
            float* at = q + ld * row(i, e);
            *at = ADD ? *at + value(acc.x[i][j][e]) : value(acc.x[i][j][e]);
          }
    }
  }
}

struct Split {
  int splits, steps;
};
// Splits of a contraction so that the tiles fill the 256 CUs, each at least 16
// steps (256 k) long.
inline Split split_of(int64_t M, int64_t N, int steps) {
  const int64_t tiles = (M + TM - 1) / TM * ((N + TN - 1) / TN);
  int64_t s = tiles >= 224 ? 1 : 256 / tiles;
  if (s > steps / 16) s = steps / 16;
  if (s < 1) s = 1;
  int per = (int)((steps + s - 1) / s);
  per = (per + 1) / 2 * 2;
  return Split{(steps + per - 1) / per, per};
}

}  // namespace pr
}  // namespace cnhip
