// Controls on logits: penalties on the tokens of a row's history, biases on listed tokens, a bit mask of allowed tokens; the row
// is stored, or its best token selected (the largest logit, or the largest of logit / temperature plus Gumbel noise).
//
//   v = l > 0 ? l / r : l r      where the token occurred in prompt or answer (r: repetition)
//   v = v - f c                  c: how often it occurred in the answer (f: frequency)
//   v = v - p                    where c > 0 (p: presence)
//   v = v + b                    b: sum of the row's biases of this token, in the order they are listed
//   v = -inf                     where the mask's bit is 0
//
// All in fp32, each step rounded on its own (no fused multiply-add), so that a selected token is the one that the same steps
// written out give. A CTA takes a row in slices of kSlice tokens and counts the history's tokens of a slice in shared memory;
// integer atomics, so the order of arrival changes nothing.
#include <math.h>
#include <math_constants.h>

#include "xpool/elem.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace controls {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;
constexpr uint32_t kInPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;

__device__ __forceinline__ uint32_t hash3(uint32_t a, uint32_t b, uint32_t c) {
  uint64_t x = (static_cast<uint64_t>(a) << 32) ^ (static_cast<uint64_t>(b) * 0x9E3779B97F4A7C15ull) ^ c;
  x ^= x >> 30;
  x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27;
  x *= 0x94D049BB133111EBull;
  x ^= x >> 31;
  return static_cast<uint32_t>(x >> 16);
}

struct Row {
  const int* history;
  int len, prompt, latest;          // latest: token of place len - 1, or -1 when it is stored
  int bias0, bias1;
  const uint32_t* mask;
  float repetition, frequency, presence, inv_t;
  bool noisy;
  uint32_t seed, step;
};

__device__ __forceinline__ Row load_row(const XpLogitArgs& a, int r) {
  const XpLogitControls& c = a.c;
  Row w;
  w.history = nullptr, w.len = 0, w.prompt = 0, w.latest = -1;
  if (c.history != nullptr) {
    const int slot = c.history_rows != nullptr ? c.history_rows[r] : r;
    if (slot >= 0 && slot < c.history_slots) {
      w.history = c.history + static_cast<size_t>(slot) * c.ld_history;
      w.len = min(max(c.lens[r], 0), c.history_cap);
      w.prompt = c.prompt_lens != nullptr ? c.prompt_lens[r] : 0;
      if (c.latest != nullptr && w.len > 0) w.latest = c.latest[r];
    }
  }
  w.bias0 = w.bias1 = 0;
  if (c.bias_starts != nullptr) {
    w.bias0 = min(max(c.bias_starts[r], 0), c.bias_total);
    w.bias1 = min(max(c.bias_starts[r + 1], w.bias0), c.bias_total);
  }
  const int m = c.mask_index != nullptr ? c.mask_index[r] : -1;
  w.mask = m >= 0 && m < c.mask_count ? c.masks + static_cast<size_t>(m) * c.ld_mask : nullptr;
  w.repetition = c.repetition != nullptr ? c.repetition[r] : 1.f;
  w.frequency = c.frequency != nullptr ? c.frequency[r] : 0.f;
  w.presence = c.presence != nullptr ? c.presence[r] : 0.f;
  const float t = a.temps != nullptr ? a.temps[r] : 0.f;
  w.noisy = t > 0.f;
  w.inv_t = w.noisy ? 1.f / t : 1.f;
  w.seed = w.noisy ? a.seeds[2 * r] : 0, w.step = w.noisy ? a.seeds[2 * r + 1] : 0;
  return w;
}

__device__ __forceinline__ float penalised(float l, uint32_t word, const Row& w) {
  const uint32_t count = word & kCount;
  if ((word & (kInPrompt | kCount)) == 0) return l;
  float v = l > 0.f ? __fdiv_rn(l, w.repetition) : __fmul_rn(l, w.repetition);
  v = __fsub_rn(v, __fmul_rn(w.frequency, static_cast<float>(count)));
  return count > 0 ? __fsub_rn(v, w.presence) : v;
}

struct Best {
  float key, value;
  int token;
  __device__ __forceinline__ Best() : key(-INFINITY), value(-INFINITY), token(0x7fffffff) {}
  __device__ __forceinline__ void offer(float k, float v, int t) {
    if (k > key || (k == key && t < token)) key = k, value = v, token = t;
  }
  __device__ __forceinline__ void warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float k = __shfl_xor_sync(0xffffffffu, key, o), v = __shfl_xor_sync(0xffffffffu, value, o);
      const int t = __shfl_xor_sync(0xffffffffu, token, o);
      offer(k, v, t);
    }
  }
};

template <typename T, typename O, bool kSelect>
__global__ void __launch_bounds__(kThreads)
logit_controls_kernel(XpLogitArgs a) {
  pdl::wait();
  pdl::release();
  __shared__ uint32_t table[kSlice];
  __shared__ float keys[kThreads / 32], vals[kThreads / 32];
  __shared__ int toks[kThreads / 32];
  const int r = blockIdx.x;
  const Row w = load_row(a, r);
  const T* row = reinterpret_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  O* out = reinterpret_cast<O*>(a.out) + static_cast<size_t>(r) * a.ld_out;
  const bool touched = w.len > 0 || w.bias1 > w.bias0;
  Best best;
  auto finish = [&](int i, float v) {
    if (w.mask != nullptr && ((w.mask[i >> 5] >> (i & 31)) & 1u) == 0) v = -CUDART_INF_F;
    if constexpr (kSelect) {
      float k = v * w.inv_t;
      if (w.noisy) {
        const float u = (static_cast<float>(hash3(w.seed, w.step, static_cast<uint32_t>(i)) >> 8) + 0.5f) * (1.f / 16777216.f);
        k -= __logf(-__logf(u));
      }
      best.offer(k, v, i);
    } else {
      elem::st(out + i, v);
    }
  };
  for (int lo = 0; lo < a.vocab; lo += kSlice) {
    const int n = min(kSlice, a.vocab - lo);
    int repeats = 0;
    if (touched) {
      for (int i = threadIdx.x; i < n; i += kThreads) table[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < w.len; i += kThreads) {
        const int id = i == w.len - 1 && w.latest >= 0 ? w.latest : w.history[i];
        if (id < lo || id >= lo + n) continue;
        if (i < w.prompt) atomicOr(&table[id - lo], kInPrompt);
        else atomicAdd(&table[id - lo], 1u);
      }
      __syncthreads();
      for (int e = w.bias0 + threadIdx.x; e < w.bias1; e += kThreads) {
        const int id = a.c.bias_ids[e];
        if (id >= lo && id < lo + n && (atomicOr(&table[id - lo], kBiased) & kBiased)) repeats = 1;
      }
      repeats = __syncthreads_or(repeats);
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t word = touched ? table[i] : 0u;
      if (word & kBiased) continue;
      finish(lo + i, penalised(elem::ld(row + lo + i), word, w));
    }
    // biased tokens: the thread of a token's first entry adds up all of them
    for (int e = w.bias0 + threadIdx.x; e < w.bias1; e += kThreads) {
      const int id = a.c.bias_ids[e];
      if (id < lo || id >= lo + n) continue;
      float sum = a.c.bias_values[e];
      if (repeats) {
        bool first = true;
        for (int f = w.bias0; f < e && first; ++f) first = a.c.bias_ids[f] != id;
        if (!first) continue;
        for (int f = e + 1; f < w.bias1; ++f)
          if (a.c.bias_ids[f] == id) sum = __fadd_rn(sum, a.c.bias_values[f]);
      }
      finish(id, __fadd_rn(penalised(elem::ld(row + id), table[id - lo], w), sum));
    }
    __syncthreads();
  }
  if (w.latest >= 0 && threadIdx.x == 0) const_cast<int*>(w.history)[w.len - 1] = w.latest;
  if constexpr (kSelect) {
    best.warp();
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) keys[warp] = best.key, vals[warp] = best.value, toks[warp] = best.token;
    __syncthreads();
    if (threadIdx.x < 32) {
      Best b;
      if (threadIdx.x < kThreads / 32) b.key = keys[threadIdx.x], b.value = vals[threadIdx.x], b.token = toks[threadIdx.x];
      b.warp();
      if (threadIdx.x == 0) {
        a.tokens[r] = b.token;
        if (a.values != nullptr) a.values[r] = b.value;
      }
    }
  }
}

}  // namespace controls
}  // namespace xpool

extern "C" int xp_logit_controls(const XpLogitArgs* a, void* stream) {
  using namespace xpool::controls;
  if (a->rows <= 0) return 0;
  if (a->vocab <= 0 || a->ld < a->vocab || (a->out != nullptr && a->ld_out < a->vocab)) return -10;
  if (a->out == nullptr && a->tokens == nullptr) return -11;
  if (a->c.history != nullptr && a->c.lens == nullptr) return -12;
  if (a->c.bias_starts != nullptr && a->c.bias_total > 0 && (a->c.bias_ids == nullptr || a->c.bias_values == nullptr)) return -12;
  if (a->temps != nullptr && a->seeds == nullptr) return -13;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  using bf16 = __nv_bfloat16;
  auto go = [&](auto kernel) { return xpool::pdl::launch(kernel, a->rows, kThreads, 0, s, 1, *a); };
  if (a->out == nullptr) {
    a->f32 ? go(logit_controls_kernel<float, float, true>) : go(logit_controls_kernel<bf16, float, true>);
  } else if (a->out_f32) {
    a->f32 ? go(logit_controls_kernel<float, float, false>) : go(logit_controls_kernel<bf16, float, false>);
  } else {
    a->f32 ? go(logit_controls_kernel<float, bf16, false>) : go(logit_controls_kernel<bf16, bf16, false>);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}
