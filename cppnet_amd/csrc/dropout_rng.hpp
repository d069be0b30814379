// The counter-based generator of dropout's masks, shared by every kernel that
// draws one, so that equal positions give equal masks whichever call asks.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace cnhip {

constexpr uint64_t kDropoutStep = 0x9E3779B97F4A7C15ull;

// The top 24 bits of splitmix64's output for the word z = seed + position * kDropoutStep.
// (Its last step, z ^= z >> 31, leaves those bits as they are.)
__device__ __forceinline__ uint32_t dropout_top24(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (uint32_t)(z >> 40);
}

// An element is kept where its 24 bits are below this: u < 1 - p for u = top24 / 2^24,
// as fp32 computes 1 - p.
inline uint32_t dropout_limit(float p) { return (uint32_t)std::ceil((1.0f - p) * 16777216.0f); }

}  // namespace cnhip
