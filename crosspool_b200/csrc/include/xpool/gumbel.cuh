// Noise of a draw: argmax_i (logit_i / T + g_i) with g_i = -log(-log u_i) draws from softmax(logits / T), in one pass and without
// normalising. u_i comes from a counter-based hash of (row seed, step, token), so the same triple always yields the same noise.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace xpool {
namespace gumbel {

__device__ __forceinline__ uint32_t hash3(uint32_t a, uint32_t b, uint32_t c) {
  uint64_t x = (static_cast<uint64_t>(a) << 32) ^ (static_cast<uint64_t>(b) * 0x9E3779B97F4A7C15ull) ^ c;
  x ^= x >> 30;
  x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27;
  x *= 0x94D049BB133111EBull;
  x ^= x >> 31;
  return static_cast<uint32_t>(x >> 16);
}

// -g_i. u is the middle of one of 2^24 even steps. That of the last one, 1 - 2^-25, is 1 in 32 bits, whose noise would be infinite: an
// unlikely token would be drawn for sure, in one of 110 draws from 151936 tokens. -log u is 2^-25 there, and above 2^-24 elsewhere.
__device__ __forceinline__ float minus_noise(uint32_t seed, uint32_t step, uint32_t token) {
  const float u = (static_cast<float>(hash3(seed, step, token) >> 8) + 0.5f) * (1.f / 16777216.f);
  return __logf(fmaxf(-__logf(u), 0x1p-25f));
}

}  // namespace gumbel
}  // namespace xpool
