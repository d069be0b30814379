// A gated linear recurrence over sequences [B, S, D], every feature of a sample
// for itself, and its backward pass.
//
//   a = sigmoid(f), w = sigmoid(i), or 1 - a without an input gate
//   h_t = a_t h_{t-1} + w_t x_t
// backward, from the last step to the first, u the gradient that a step hands to
// the state before it:
//   g_t = dh_t + u_{t+1},  u_t = a_t g_t,
//   dx = w g,  df = a (1 - a) g (h_{t-1} - x_t) (with an input gate: a (1 - a) g
//   h_{t-1}, di = w (1 - w) g x).
//
// Both directions are the same problem: maps s -> a s + b one after the other.
// Two maps in a row are a map again, so runs of steps are joined in any grouping:
// a lane joins its own steps, the wave scans its lanes, the waves of a block pass
// their totals through LDS, and each lane then runs its steps again from the state
// that enters it.  The inputs are read once.
//
// The factor of a map is held in two floats (hi + lo).  A gate that remembers has
// 1 - a far below 1, and a in one float keeps 1 - a to no more than 2^-25 of 1: a
// gate of f = 8 would forget a ten-thousandth too much or too little, every step
// alike.
//
// Bound by memory: 2 x 32768 steps of width 1024 take 185 us forward (805 MB, 4.4 TB/s)
// and 344 back (1.6 GB, 4.7 TB/s), where a large copy moves 4.9; 32 x 256 of width 512
// 12.1 and 18.4 (4.2 and 5.5 TB/s, in part from the caches).  The forward's 79 vector
// instructions for 64 steps are 108 of its 185 us.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "act_math.hpp"
#include "common.hpp"

namespace cnhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMostWaves = 16;

// s -> (p + l) s + y
struct Map {
  float p, l, y;
};
__device__ __forceinline__ Map identity() { return Map{1.f, 0.f, 0.f}; }
__device__ __forceinline__ float apply(const Map& m, float s) { return fmaf(m.p, s, fmaf(m.l, s, m.y)); }
// `first`, then `next`
__device__ __forceinline__ Map join(const Map& first, const Map& next) {
  Map r;
  r.p = first.p * next.p;
  r.l = fmaf(first.p, next.p, -r.p) + fmaf(first.p, next.l, first.l * next.p);
  r.y = apply(next, first.y);
  return r;
}

// sigmoid(z) and 1 - sigmoid(z), each to its own relative precision, and what the
// rounding of the first leaves of 1 - the second.
__device__ __forceinline__ void gate(float z, float& on, float& off, float& rest) {
  // (beyond 200 nothing is left of e; infinities are gates that keep or drop everything)
  const float e = exp_acc(-fminf(fabsf(z), 200.f)), r = __builtin_amdgcn_rcpf(1.f + e);
  const float small = e * r;
  const float large = 1.f - small;  // 1 - small is closer to it than r
  on = z >= 0.f ? large : small;
  off = z >= 0.f ? small : large;
  rest = z >= 0.f ? (1.f - large) - small : 0.f;
  if (z != z) on = off = z;
}

struct RecArgs {
  const float *x, *f, *i, *h0, *h, *dh, *dh_last;
  float *out, *last;       // forward: h, h_last
  float *dx, *df, *di, *dh0;
  const int32_t* len;
  int64_t B, S, D, chains;
  int64_t block0;          // of this launch, of all the blocks
  int waves;               // that share a chain's steps (of a group of samples' in the reference's row order)
  int lanes;               // V with short sequences: lanes a chain takes
  int segments;            // pieces of the steps, in blocks of their own
  int64_t segment;         // their steps
  Map* part;               // [segment][chain]
  float* start;            // [chain]: the state before the first step
};

__device__ __forceinline__ float shift_dpp(float old, float x, int which) {
  const int o = __builtin_bit_cast(int, old), v = __builtin_bit_cast(int, x);
  int r;
  switch (which) {  // row_shr 1, 2, 4, 8, row_bcast 15 and 31, wave_shr 1
    case 0: r = __builtin_amdgcn_update_dpp(o, v, 0x111, 0xF, 0xF, false); break;
    case 1: r = __builtin_amdgcn_update_dpp(o, v, 0x112, 0xF, 0xF, false); break;
    case 2: r = __builtin_amdgcn_update_dpp(o, v, 0x114, 0xF, 0xF, false); break;
    case 3: r = __builtin_amdgcn_update_dpp(o, v, 0x118, 0xF, 0xF, false); break;
    case 4: r = __builtin_amdgcn_update_dpp(o, v, 0x142, 0xA, 0xF, false); break;
    case 5: r = __builtin_amdgcn_update_dpp(o, v, 0x143, 0xC, 0xF, false); break;
    default: r = __builtin_amdgcn_update_dpp(o, v, 0x138, 0xF, 0xF, false); break;
  }
  return __builtin_bit_cast(float, r);
}
// The map of the lanes before this one, by one step of the scan over the whole wave.
__device__ __forceinline__ Map earlier(const Map& m, int which) {
  return Map{shift_dpp(1.f, m.p, which), shift_dpp(0.f, m.l, which), shift_dpp(0.f, m.y, which)};
}
// The map `o` lanes before; the identity for lanes at `at` < o of their chain.
__device__ __forceinline__ Map earlier(const Map& m, int o, int at) {
  const Map r{__shfl_up(m.p, o, 64), __shfl_up(m.l, o, 64), __shfl_up(m.y, o, 64)};
  return at >= o ? r : identity();
}
__device__ __forceinline__ Map from_lane(const Map& m, int lane) {
  return Map{__shfl(m.p, lane, 64), __shfl(m.l, lane, 64), __shfl(m.y, lane, 64)};
}

// How the lanes of a wave take the steps.
//   kRun: the steps of a chain lie side by side (rows by sample, or one sample).
//     A lane takes 4 in a row, U times 256 steps further.
//   kShort: the same for sequences of up to 128 steps; a wave takes several chains.
//   kStrided: rows in the reference's order, a step's samples side by side.  The lanes
//     of a wave take the samples (up to 64) of one feature and, of fewer than 33, 4
//     steps in a row of each, U times.  A load then reads every fourth step's line, and
//     the four loads read them whole (a step a lane, so that each load runs along
//     memory, joins maps across lanes for every step and not for every fourth: 5 x
//     1001, width 333, with its gradients, 61 us for 39).
enum Layout { kRun, kShort, kStrided };

// PASS 0: everything.  Where few chains have many steps these are cut in segments:
// PASS 1 leaves each segment's map, PASS 2 runs it from the segments before.
template <Layout LAY, bool BWD, bool IG, int U, int PASS>
__global__ void __launch_bounds__(1024) recurrence_kernel(RecArgs a) {
  constexpr int E = 4;
  __shared__ Map totals[2][kMostWaves][LAY == kStrided ? 64 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int seat = wave % a.waves;  // of the waves that share a chain
  const int64_t team = (a.block0 + blockIdx.x) * ((blockDim.x >> 6) / a.waves) + wave / a.waves;
  const int64_t BS = a.B * a.S;

  // this lane's chain (c = b + B d), its place among the wave's lanes
  int64_t c, b;
  int at, width;  // kStrided: step of the wave's `width`; else lane of the chain's `width`
  bool mine;
  if constexpr (LAY == kRun) {
    c = team;
    mine = c < a.chains;
    at = lane;
    width = 64;
  } else if constexpr (LAY == kShort) {
    c = team * (64 / a.lanes) + lane / a.lanes;
    mine = c < a.chains;
    at = lane % a.lanes;
    width = a.lanes;
  } else {
    const int64_t groups = (a.B + 63) / 64, d = team / groups;
    const int n = a.B < 64 ? (int)a.B : 64;
    width = 64 / n;
    at = lane / n;
    b = (team % groups) * 64 + lane % n;
    c = b + a.B * d;
    mine = d < a.D && b < a.B && at < width;
  }
  const int stride = LAY == kStrided ? (int)(a.B < 64 ? a.B : 64) : 1;  // lanes from one step to the next
  if (!mine) c = at = 0;  // reads what exists, writes nothing
  if (LAY != kStrided) b = c % a.B;
  else if (!mine) b = 0;
  const int64_t base = LAY == kStrided ? b + BS * (c / a.B) : a.S * c;  // the chain's first step
  const int64_t step = LAY == kStrided ? a.B : 1;
  int64_t len = a.S;
  if (a.len) {
    const int32_t n = a.len[b];
    len = n < 0 ? 0 : n < a.S ? n : a.S;
  }

  const int seg = PASS ? (int)blockIdx.y : 0;
  const int64_t q_begin = PASS ? seg * a.segment : 0;
  const int64_t q_end = PASS ? (q_begin + a.segment < a.S ? q_begin + a.segment : a.S) : a.S;
  // steps of a wave and of all that share a chain, in a round
  const int span = U * E * width;
  const int64_t round = (int64_t)span * a.waves;

  float state = 0.f;  // what enters the round
  if constexpr (PASS == 2) {
    if (mine) {
      state = a.start[c];
      for (int g = 0; g < seg; ++g) state = apply(a.part[(int64_t)g * a.chains + c], state);
    }
  } else {
    const float* s0 = BWD ? a.dh_last : a.h0;
    if (s0 && mine) state = s0[c];
    if (PASS == 1 && seg == 0 && mine && seat == 0 && at == 0) a.start[c] = state;
  }

  struct Raw {
    float f[U][E], x[U][E], i[U][E], hp[U][E], dh[U][E];
  };
  // position q0 + e in the order of the maps is step t
  auto first_q = [&](int64_t r0, int u) { return r0 + (int64_t)seat * span + (u * width + at) * E; };
  // Whether all of the wave's steps of a round exist and are within their lengths.  Its
  // loads then go out one after the other; behind tests of their own each would be
  // waited for.
  auto is_whole = [&](int64_t r0) {
    const int64_t w0 = r0 + (int64_t)seat * span;
    return w0 + span <= q_end && __all(!mine || (BWD ? a.S - w0 <= len : w0 + span <= len));
  };
  auto load = [&](int64_t r0, Raw& v, auto whole_tag) {
    constexpr bool WHOLE = decltype(whole_tag)::value;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t q0 = first_q(r0, u);
      // the steps of these positions, [lo, lo + E)
      const int64_t lo = BWD ? a.S - E - q0 : q0;
      const bool any = WHOLE || (mine && q0 < q_end && lo < len);
      auto get = [&](const float* p, float (&to)[E], auto back_tag) {
        constexpr int back = decltype(back_tag)::value;
        if (LAY != kStrided && (WHOLE || (any && q0 + 4 <= a.S && lo >= back))) {
          // (the state before step 0 is not read from here: the first chain's would lie before h)
          const int64_t o = base + lo - back;
          const bool edge = back && o < 0;
          const f32x4 w = *reinterpret_cast<const f32x4u*>(p + (edge ? 0 : o));
#pragma unroll
          for (int e = 0; e < E; ++e) to[e] = !BWD ? w[e] : edge && e + 1 < E ? w[E - 2 - e] : w[E - 1 - e];
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int64_t t = BWD ? a.S - 1 - (q0 + e) : q0 + e, o = base + step * (t - back);
            if (WHOLE) to[e] = p[back && o < 0 ? 0 : o];
            else to[e] = any && t >= back && t < a.S ? p[o] : 0.f;
          }
        }
      };
      constexpr std::integral_constant<int, 0> now;
      constexpr std::integral_constant<int, 1> before;
      get(a.f, v.f[u], now);
      if (!BWD || PASS != 1) get(a.x, v.x[u], now);
      if (IG && (!BWD || PASS != 1)) get(a.i, v.i[u], now);
      if constexpr (BWD) {
        get(a.dh, v.dh[u], now);
        if (PASS != 1) get(a.h, v.hp[u], before);
      }
    }
  };

  Raw raw;
  bool whole_now = false, whole_next = false;
  auto load_any = [&](int64_t r0) {
    whole_next = is_whole(r0);
    if (whole_next) load(r0, raw, std::true_type{});
    else load(r0, raw, std::false_type{});
  };
  load_any(q_begin);
  Map whole = identity();  // PASS 1: of the rounds so far
  const float first = BWD && PASS != 1 && a.h0 && mine ? a.h0[c] : 0.f;
  int parity = 0;
  for (int64_t r0 = q_begin; r0 < q_end; r0 += round, parity ^= 1) {
    whole_now = whole_next;
    // forward: b = w x.  backward: b = dh, entered before the factor
    float p[U][E], l[U][E], y[U][E], w[U][E], off[U][E], wo[U][E], x[U][E], hp[U][E];
    Map m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = identity();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t q = first_q(r0, u) + e, t = BWD ? a.S - 1 - q : q;
        const bool in = whole_now || (q < q_end && t < len);
        gate(raw.f[u][e], p[u][e], off[u][e], l[u][e]);
        if (IG) {
          float none;
          gate(raw.i[u][e], w[u][e], wo[u][e], none);
        } else {
          w[u][e] = off[u][e];
        }
        x[u][e] = raw.x[u][e];
        if constexpr (BWD) {
          hp[u][e] = raw.hp[u][e];
          y[u][e] = in ? raw.dh[u][e] : 0.f;
        } else {
          y[u][e] = in ? w[u][e] * x[u][e] : 0.f;
        }
        p[u][e] = in ? p[u][e] : 1.f;
        l[u][e] = in ? l[u][e] : 0.f;
        if constexpr (BWD) {
          const float by = fmaf(p[u][e], y[u][e], l[u][e] * y[u][e]);
          m[u] = join(m[u], Map{p[u][e], l[u][e], by});
        } else {
          m[u] = join(m[u], Map{p[u][e], l[u][e], y[u][e]});
        }
      }
    }
    if (r0 + round < q_end) load_any(r0 + round);
    // m: of the lane's own steps -> of the chain's lanes up to this one; before: without it
    Map before[U], total[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (LAY == kRun) {
#pragma unroll
        for (int k = 0; k < 6; ++k) m[u] = join(earlier(m[u], k), m[u]);
        before[u] = earlier(m[u], 6);
        total[u] = from_lane(m[u], 63);
      } else if constexpr (LAY == kShort) {
        for (int o = 1; o < width; o <<= 1) m[u] = join(earlier(m[u], o, at), m[u]);
        before[u] = earlier(m[u], 1, at);
        total[u] = from_lane(m[u], lane - at + width - 1);
      } else {
        for (int o = 1; o < width; o <<= 1) m[u] = join(earlier(m[u], o * stride, at * stride), m[u]);
        before[u] = width > 1 ? earlier(m[u], stride, at * stride) : identity();
        total[u] = width > 1 ? from_lane(m[u], (lane % stride + (width - 1) * stride) & 63) : m[u];
      }
    }
    Map wave_map = total[0];
#pragma unroll
    for (int u = 1; u < U; ++u) wave_map = join(wave_map, total[u]);
    float enter = state;
    if (a.waves > 1) {
      const int slot = LAY == kStrided ? lane : 0;
      if (LAY == kStrided || lane == 0) totals[parity][wave][slot] = wave_map;
      __syncthreads();
      Map all = identity();
      for (int s = 0; s < a.waves; ++s) {
        if (PASS == 1) {
          all = join(all, totals[parity][wave - seat + s][slot]);
          continue;
        }
        if (s == seat) enter = state;
        state = apply(totals[parity][wave - seat + s][slot], state);
      }
      if (PASS == 1) whole = join(whole, all);
    } else {
      if (PASS == 1) whole = join(whole, wave_map);
      else state = apply(wave_map, state);
    }
    if constexpr (PASS == 1) continue;
    auto finish = [&](auto whole_tag) {
      constexpr bool WHOLE = decltype(whole_tag)::value;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float s = apply(before[u], enter);
        enter = apply(total[u], enter);
        const int64_t q0 = first_q(r0, u);
        float o0[E], o1[E], o2[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t q = q0 + e, t = BWD ? a.S - 1 - q : q;
          const bool in = WHOLE || t < len;
          if constexpr (BWD) {
            const float g = y[u][e] + s;
            const float prev = t == 0 ? first : hp[u][e];
            const float df = p[u][e] * off[u][e] * g;
            o0[e] = in ? w[u][e] * g : 0.f;
            o1[e] = in ? df * (IG ? prev : prev - x[u][e]) : 0.f;
            if (IG) o2[e] = in ? w[u][e] * wo[u][e] * g * x[u][e] : 0.f;
            s = fmaf(p[u][e], g, l[u][e] * g);
          } else {
            s = fmaf(p[u][e], s, fmaf(l[u][e], s, y[u][e]));
            o0[e] = in ? s : 0.f;
          }
        }
        if (!mine || (!WHOLE && q0 >= q_end)) continue;
        auto put = [&](float* to, const float (&v)[E]) {
          if (LAY != kStrided && (WHOLE || q0 + 4 <= q_end)) {
            f32x4 w4;
#pragma unroll
            for (int e = 0; e < E; ++e) w4[BWD ? E - 1 - e : e] = v[e];
            *reinterpret_cast<f32x4u*>(to + base + (BWD ? a.S - 4 - q0 : q0)) = w4;
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (WHOLE || q0 + e < q_end) to[base + step * (BWD ? a.S - 1 - (q0 + e) : q0 + e)] = v[e];
          }
        };
        if constexpr (BWD) {
          put(a.dx, o0);
          put(a.df, o1);
          if (IG) put(a.di, o2);
        } else {
          put(a.out, o0);
        }
      }
    };
    if (whole_now) finish(std::true_type{});
    else finish(std::false_type{});
  }
  if (!mine || seat || at) return;
  if (PASS == 1) {
    a.part[(int64_t)seg * a.chains + c] = whole;
    return;
  }
  float* last = BWD ? a.dh0 : a.last;
  if (last && q_end == a.S) last[c] = state;
}

template <Layout LAY, bool BWD, bool IG, int U>
int launch(RecArgs& a, int64_t blocks, int threads, hipStream_t st, const char* who) {
  if (a.segments == 1) {
    // a grid has fewer than 2^32 threads
    constexpr int64_t most = (int64_t)1 << 21;
    for (; a.block0 < blocks; a.block0 += most) {
      const int64_t left = blocks - a.block0;
      hipLaunchKernelGGL((recurrence_kernel<LAY, BWD, IG, U, 0>), dim3((unsigned)(left < most ? left : most)),
                         dim3(threads), 0, st, a);
      CNHIP_TRY(check_launch(who));
    }
    return CNHIP_OK;
  }
  const dim3 grid((unsigned)blocks, (unsigned)a.segments);
  if constexpr (LAY != kShort && (BWD || U == 2)) {  // (the forward's U = 1 is for short sequences)
    hipLaunchKernelGGL((recurrence_kernel<LAY, BWD, IG, U, 1>), grid, dim3(threads), 0, st, a);
    CNHIP_TRY(check_launch(who));
    hipLaunchKernelGGL((recurrence_kernel<LAY, BWD, IG, U, 2>), grid, dim3(threads), 0, st, a);
  }
  return check_launch(who);
}

template <bool BWD, bool IG>
int run(RecArgs& a, int rows, hipStream_t st, const char* who) {
  a.chains = a.B * a.D;
  const bool side = rows == CNHIP_ROWS_BY_SAMPLE || a.B == 1 || a.S == 1;  // a chain's steps lie side by side
  a.waves = a.segments = 1;
  a.lanes = 64;
  a.segment = a.S;
  if (side && a.S <= 128) {
    a.lanes = 1;
    while (4 * a.lanes < a.S) a.lanes *= 2;
    const int64_t waves = (a.chains + 64 / a.lanes - 1) / (64 / a.lanes), blocks = (waves + 3) / 4;
    return launch<kShort, BWD, IG, 1>(a, blocks, 256, st, who);
  }
  // Teams: what one wave (or the waves that share the steps) takes.  Their waves are as
  // many as are resident with all teams (a CU holds 16 of these kernels) and as there are
  // steps for, and no more than the rounds that this makes need.
  const int64_t teams = side ? a.chains : a.D * ((a.B + 63) / 64);
  const int width = side ? 64 : a.B > 32 ? 1 : (int)(64 / a.B);
  const int u = BWD || (side && a.S <= 256) ? 1 : 2;
  const int64_t span = (int64_t)u * 4 * width;
  const int64_t per_cu = (teams + 255) / 256, most = per_cu < kMostWaves ? kMostWaves / per_cu : 1;
  const int64_t rounds = (a.S + span * most - 1) / (span * most);
  a.waves = (int)((a.S + span * rounds - 1) / (span * rounds));
  const int64_t full = span * kMostWaves;
  // Half the chip would idle: at most 128 blocks, so that from 65 teams on, or below twice
  // the steps of a block of all waves, one block still takes a chain's steps from end to end.
  if (teams < 128 && a.S >= 2 * full) {
    a.waves = kMostWaves;
    int64_t n = 128 / teams;
    if (n > a.S / full) n = a.S / full;
    a.segment = ((a.S + n - 1) / n + full - 1) / full * full;
    a.segments = (int)((a.S + a.segment - 1) / a.segment);
  }
  const int per = a.waves < 4 ? 4 / a.waves : 1, block_waves = per * a.waves;
  const int64_t blocks = (teams + per - 1) / per;
  if (a.segments > 1) {
    void* ws = nullptr;
    const size_t parts = (size_t)a.segments * (size_t)a.chains * sizeof(Map);
    CNHIP_TRY(scratch(st, kScratchLayer, parts + (size_t)a.chains * sizeof(float), &ws, who));
    a.part = static_cast<Map*>(ws);
    a.start = reinterpret_cast<float*>(static_cast<char*>(ws) + parts);
  }
  if (!side) return launch<kStrided, BWD, IG, BWD ? 1 : 2>(a, blocks, 64 * block_waves, st, who);
  if constexpr (!BWD) {
    if (u == 2) return launch<kRun, BWD, IG, 2>(a, blocks, 64 * block_waves, st, who);
  }
  return launch<kRun, BWD, IG, 1>(a, blocks, 64 * block_waves, st, who);
}

int check_shape(int64_t B, int64_t S, int64_t D, int rows, const char* who) {
  CNHIP_REQUIRE(B > 0 && S > 0 && D > 0, "%s: bad shape B=%lld S=%lld D=%lld", who, (long long)B, (long long)S,
                (long long)D);
  CNHIP_REQUIRE(rows == CNHIP_ROWS_REF || rows == CNHIP_ROWS_BY_SAMPLE, "%s: bad row order %d", who, rows);
  CNHIP_REQUIRE(B < ((int64_t)1 << 30) && S < ((int64_t)1 << 30) && D < ((int64_t)1 << 30) &&
                    B * D < ((int64_t)1 << 40) && S < ((int64_t)1 << 60) / (B * D),
                "%s: too large", who);
  return CNHIP_OK;
}

}  // namespace
}  // namespace cnhip

extern "C" {

int cnhip_linear_recurrence_forward(const float* x, const float* f, const float* i, const float* h0, float* h,
                                    float* h_last, int64_t B, int64_t S, int64_t D, const int32_t* seq_len, int rows,
                                    cnhip_stream_t stream) {
  const char* who = "cnhip_linear_recurrence_forward";
  CNHIP_TRY(cnhip::check_shape(B, S, D, rows, who));
  CNHIP_REQUIRE(x && f && h, "%s: NULL pointer", who);
  cnhip::RecArgs a{};
  a.x = x;
  a.f = f;
  a.i = i;
  a.h0 = h0;
  a.out = h;
  a.last = h_last;
  a.len = seq_len;
  a.B = B;
  a.S = S;
  a.D = D;
  const hipStream_t st = cnhip::as_stream(stream);
  cnhip::HbmTimer timer("recurrence_kernel", (i ? 16.0 : 12.0) * (double)B * (double)S * (double)D, st);
  return i ? cnhip::run<false, true>(a, rows, st, who) : cnhip::run<false, false>(a, rows, st, who);
}

int cnhip_linear_recurrence_backward(const float* x, const float* f, const float* i, const float* h0, const float* h,
                                     const float* dh, const float* dh_last, float* dx, float* df, float* di, float* dh0,
                                     int64_t B, int64_t S, int64_t D, const int32_t* seq_len, int rows,
                                     cnhip_stream_t stream) {
  const char* who = "cnhip_linear_recurrence_backward";
  CNHIP_TRY(cnhip::check_shape(B, S, D, rows, who));
  CNHIP_REQUIRE(x && f && h && dh && dx && df, "%s: NULL pointer", who);
  CNHIP_REQUIRE(!i == !di, "%s: di goes with i", who);
  cnhip::RecArgs a{};
  a.x = x;
  a.f = f;
  a.i = i;
  a.h0 = h0;
  a.h = h;
  a.dh = dh;
  a.dh_last = dh_last;
  a.dx = dx;
  a.df = df;
  a.di = di;
  a.dh0 = dh0;
  a.len = seq_len;
  a.B = B;
  a.S = S;
  a.D = D;
  const hipStream_t st = cnhip::as_stream(stream);
  cnhip::HbmTimer timer("recurrence_backward_kernel", (i ? 32.0 : 24.0) * (double)B * (double)S * (double)D, st);
  return i ? cnhip::run<true, true>(a, rows, st, who) : cnhip::run<true, false>(a, rows, st, who);
}

}  // extern "C"
