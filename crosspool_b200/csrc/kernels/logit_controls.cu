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
// written out give. Bound by reading the logits once (and writing them once): a CTA takes a row, or a cluster of up to eight shares
// one while rows are few, 16 bytes a load. Only few tokens of a row are touched by its history and biases, so the stream does no
// look-ups: the CTA first marks them in a bitmap in shared memory (a bit per token of its share) and counts their occurrences in a
// hash table beside it; the stream passes marked tokens over (the mask's bits are read beside the logits), and the table's tokens
// are done at the end, when their logits are in the L2. Integer atomics, so the order of arrival changes nothing. A history of more
// different tokens than the table holds is counted range by range of the vocabulary.
#include <math.h>
#include <math_constants.h>

#include <cooperative_groups.h>

#include <utility>

#include "xpool/elem.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace controls {

constexpr int kSlots = 4096;                       // tokens of a share that can be counted at once: kSlots - kRoom
constexpr int kRoom = 1024;                        // slots left so that a search ends: one per thread of the largest CTA
constexpr uint32_t kEmpty = 0xffffffffu;
constexpr uint32_t kInPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;
constexpr int kMaxRanks = 8;
constexpr int kUnit = 1024;                        // shares are multiples of so many tokens

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
  __device__ __forceinline__ int token(int i) const { return i == len - 1 && latest >= 0 ? latest : history[i]; }
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

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Occurrences of marked tokens, found by linear search from a hashed place.
struct Table {
  uint32_t* keys;
  uint32_t* words;
  __device__ __forceinline__ static int place(uint32_t id) { return static_cast<int>((id * 2654435761u) >> 20); }
  // the slot of a token, which is entered where it is not there; the caller keeps kRoom slots empty
  __device__ __forceinline__ int enter(uint32_t id, bool& is_new) const {
    for (int s = place(id);; s = (s + 1) & (kSlots - 1)) {
      const uint32_t k = atomicCAS(&keys[s], kEmpty, id);
      if (k == kEmpty || k == id) {
        is_new = k == kEmpty;
        return s;
      }
    }
  }
  __device__ __forceinline__ uint32_t word(uint32_t id) const {
    for (int s = place(id);; s = (s + 1) & (kSlots - 1))
      if (keys[s] == id) return words[s];
  }
};

template <typename T, typename O, bool kSelect, int kThreads>
__global__ void __launch_bounds__(kThreads)
logit_controls_kernel(XpLogitArgs a, int wide, int ranks, int share) {
  namespace cg = cooperative_groups;
  constexpr int N = 16 / sizeof(T), kWarps = kThreads / 32;
  static_assert(kThreads <= kRoom, "a search may not end");
  __shared__ float keys_s[kMaxRanks * kWarps], vals_s[kMaxRanks * kWarps];
  __shared__ int toks_s[kMaxRanks * kWarps];
  __shared__ int entered, repeats;
  extern __shared__ __align__(16) uint32_t dyn[];
  // the first CTA's shared memory is written once that CTA is known to have started
  auto started = cg::this_cluster().barrier_arrive();
  pdl::wait();
  pdl::release();
  const int rank = blockIdx.x % ranks, r = blockIdx.x / ranks;
  const int lo = min(rank * share, a.vocab), hi = min(lo + share, a.vocab), n = hi - lo;
  const Row w = load_row(a, r);
  const T* row = reinterpret_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  O* out = reinterpret_cast<O*>(a.out) + static_cast<size_t>(r) * a.ld_out;
  const bool touched = w.len > 0 || w.bias1 > w.bias0;
  Table table{dyn, dyn + kSlots};
  uint32_t* marks = dyn + 2 * kSlots;              // a bit per token of the share
  Best best;
  auto key_of = [&](float v, int i) {
    float k = v * w.inv_t;
    if (w.noisy) {
      const float u = (static_cast<float>(hash3(w.seed, w.step, static_cast<uint32_t>(i)) >> 8) + 0.5f) * (1.f / 16777216.f);
      k -= __logf(-__logf(u));
    }
    return k;
  };

  // ---- marks and counts of the tokens that the controls touch
  // tokens [t0, t1): returns whether they found room
  auto count = [&](int t0, int t1, bool mark) {
    if (threadIdx.x == 0) entered = 0, repeats = 0;
    for (int i = threadIdx.x * 4; i < kSlots; i += kThreads * 4) {
      *reinterpret_cast<uint4*>(table.keys + i) = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
      *reinterpret_cast<uint4*>(table.words + i) = make_uint4(0, 0, 0, 0);
    }
    if (mark)
      for (int i = threadIdx.x; i < (n + 31) / 32; i += kThreads) marks[i] = 0;
    __syncthreads();
    bool full = false;
    auto enter = [&](int id, uint32_t what) -> uint32_t {
      if (mark) atomicOr(&marks[(id - lo) >> 5], 1u << ((id - lo) & 31));
      if (full || *reinterpret_cast<volatile int*>(&entered) > kSlots - kRoom) {
        full = true;
        return 0u;
      }
      bool is_new;
      const int s = table.enter(static_cast<uint32_t>(id), is_new);
      if (is_new) atomicAdd(&entered, 1);
      return what == 1u ? atomicAdd(&table.words[s], 1u) : atomicOr(&table.words[s], what);
    };
#pragma unroll 4
    for (int i = threadIdx.x; i < w.len; i += kThreads) {
      const int id = w.token(i);
      if (id >= t0 && id < t1) enter(id, i < w.prompt ? kInPrompt : 1u);
    }
    for (int e = w.bias0 + threadIdx.x; e < w.bias1; e += kThreads) {
      const int id = a.c.bias_ids[e];
      if (id >= t0 && id < t1 && (enter(id, kBiased) & kBiased)) repeats = 1;
    }
    return __syncthreads_or(full) == 0;
  };
  const bool fits = !touched || count(lo, hi, true);

  // ---- the stream: tokens without marks
  auto stream = [&](int i0, const T (&v)[N], O (&o)[N]) {
    uint32_t skip = 0u, allowed = ~0u;
    const uint32_t ones = (1u << N) - 1u;
    if (touched) skip = marks[(i0 - lo) >> 5] >> ((i0 - lo) & 31) & ones;
    if (w.mask != nullptr) allowed = w.mask[i0 >> 5] >> (i0 & 31);
    if constexpr (kSelect) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = as_float(v[j]);
      if (touched || w.mask != nullptr) {
        const uint32_t use = allowed & ~skip;
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = use >> j & 1u ? f[j] : -CUDART_INF_F;
      }
      if (w.noisy) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!(skip >> j & 1u)) best.offer(key_of(f[j], i0 + j), f[j], i0 + j);
      } else {
        float top = f[0];
#pragma unroll
        for (int j = 1; j < N; ++j) top = fmaxf(top, f[j]);
        if (top > best.key) {
#pragma unroll
          for (int j = N - 1; j >= 0; --j)
            if (f[j] == top) best.token = i0 + j;
          best.key = best.value = top;
        } else if (best.token == 0x7fffffff) {       // nothing but -inf so far: the lowest token counts
#pragma unroll
          for (int j = N - 1; j >= 0; --j)
            if (!(skip >> j & 1u)) best.token = i0 + j;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float f = (allowed | skip) >> j & 1u ? as_float(v[j]) : -CUDART_INF_F;      // marked tokens stay as they are for now
        elem::st(o + j, f);
      }
    }
  };
  const int whole = wide ? n / N : 0;
#pragma unroll 4
  for (int c = threadIdx.x; c < whole; c += kThreads) {
    __align__(16) T v[N];
    __align__(16) O o[N];
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(row + lo + c * N);
    stream(lo + c * N, v, o);
    if constexpr (!kSelect) {
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(O)) * N / 16; ++j) reinterpret_cast<uint4*>(out + lo + c * N)[j] = reinterpret_cast<const uint4*>(o)[j];
      if constexpr (sizeof(O) * N == 8) *reinterpret_cast<uint2*>(out + lo + c * N) = *reinterpret_cast<const uint2*>(o);
    }
  }
  for (int i = lo + whole * N + threadIdx.x; i < hi; i += kThreads) {
    const bool skip = touched && marks[(i - lo) >> 5] >> ((i - lo) & 31) & 1u;
    const bool allowed = w.mask == nullptr || w.mask[i >> 5] >> (i & 31) & 1u;
    const float f = as_float(row[i]), v = allowed || skip ? f : -CUDART_INF_F;
    if constexpr (kSelect) {
      if (!skip) best.offer(key_of(v, i), v, i);
    } else {
      elem::st(out + i, v);
    }
  }

  // ---- marked tokens
  auto finish = [&](int i, float v) {
    if (w.mask != nullptr && ((w.mask[i >> 5] >> (i & 31)) & 1u) == 0) v = -CUDART_INF_F;
    if constexpr (kSelect) best.offer(key_of(v, i), v, i);
    else elem::st(out + i, v);
  };
  auto marked = [&](int t0, int t1) {
    for (int s = threadIdx.x; s < kSlots; s += kThreads) {
      const uint32_t id = table.keys[s], word = table.words[s];
      if (id != kEmpty && !(word & kBiased)) finish(static_cast<int>(id), penalised(as_float(row[id]), word, w));
    }
    // biased tokens: the thread of a token's first entry adds up all of them
    for (int e = w.bias0 + threadIdx.x; e < w.bias1; e += kThreads) {
      const int id = a.c.bias_ids[e];
      if (id < t0 || id >= t1) continue;
      float sum = a.c.bias_values[e];
      if (repeats) {
        bool first = true;
        for (int f = w.bias0; f < e && first; ++f) first = a.c.bias_ids[f] != id;
        if (!first) continue;
        for (int f = e + 1; f < w.bias1; ++f)
          if (a.c.bias_ids[f] == id) sum = __fadd_rn(sum, a.c.bias_values[f]);
      }
      finish(id, __fadd_rn(penalised(as_float(row[id]), table.word(static_cast<uint32_t>(id)), w), sum));
    }
  };
  if (touched) {
    if constexpr (!kSelect) __syncthreads();         // marked tokens have been stored as they were
    if (fits) {
      marked(lo, hi);
    } else {
      // more tokens than the table holds: ranges of the vocabulary that cannot have more, one after the other
      for (int t0 = lo; t0 < hi; t0 += kSlots - kRoom) {
        const int t1 = min(t0 + kSlots - kRoom, hi);
        __syncthreads();
        count(t0, t1, false);
        marked(t0, t1);
      }
    }
  }
  if (rank == 0 && w.latest >= 0 && threadIdx.x == 0) const_cast<int*>(w.history)[w.len - 1] = w.latest;
  cg::this_cluster().barrier_wait(std::move(started));
  if constexpr (kSelect) {
    best.warp();
    if ((threadIdx.x & 31) == 0) {
      const int slot = rank * kWarps + (threadIdx.x >> 5);
      cg::this_cluster().map_shared_rank(keys_s, 0)[slot] = best.key;
      cg::this_cluster().map_shared_rank(vals_s, 0)[slot] = best.value;
      cg::this_cluster().map_shared_rank(toks_s, 0)[slot] = best.token;
    }
    cg::this_cluster().sync();
    if (rank != 0 || threadIdx.x >= 32) return;
    Best b;
    for (int i = threadIdx.x; i < ranks * kWarps; i += 32) b.offer(keys_s[i], vals_s[i], toks_s[i]);
    b.warp();
    if (threadIdx.x == 0) {
      a.tokens[r] = b.token;
      if (a.values != nullptr) a.values[r] = b.value;
    }
  }
}

template <auto kernel, int kThreads>
static int go(const XpLogitArgs& a, int wide, int ranks, int share, int smem, cudaStream_t s) {
  static uint64_t allowed = 0;                       // devices on which the kernel may have the shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -21;
  if ((allowed >> (dev & 63) & 1) == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kSlots * 4 + XP_LOGIT_VOCAB / 8) != cudaSuccess) return -21;
    allowed |= 1ull << (dev & 63);
  }
  pdl::launch(kernel, static_cast<unsigned>(a.rows) * ranks, kThreads, smem, s, ranks, a, wide, ranks, share);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}

template <int kThreads>
static int launch(const XpLogitArgs& a, int ranks, cudaStream_t s) {
  using bf16 = __nv_bfloat16;
  const int es = a.f32 ? 4 : 2, eo = a.out == nullptr ? 16 : a.out_f32 ? 4 : 2;
  auto aligned = [](const void* p, int64_t ld, int e) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * e % 16 == 0; };
  const int wide = aligned(a.logits, a.ld, es) && aligned(a.out, a.out == nullptr ? 0 : a.ld_out, eo);
  const int share = ((a.vocab + ranks - 1) / ranks + kUnit - 1) / kUnit * kUnit;
  const int smem = 2 * kSlots * 4 + (share + 31) / 32 * 4;
  if (a.out == nullptr) return a.f32 ? go<logit_controls_kernel<float, float, true, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
                                     : go<logit_controls_kernel<bf16, float, true, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
  if (a.out_f32) return a.f32 ? go<logit_controls_kernel<float, float, false, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
                              : go<logit_controls_kernel<bf16, float, false, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
  return a.f32 ? go<logit_controls_kernel<float, bf16, false, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
               : go<logit_controls_kernel<bf16, bf16, false, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
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
  if (a->vocab > XP_LOGIT_VOCAB || a->rows > (1 << 27)) return -14;
  int ranks = a->rows <= 32 ? 8 : a->rows <= 256 ? 4 : 2;
  while (ranks > 1 && a->vocab / ranks < 4 * kUnit) ranks >>= 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->vocab / ranks <= 4 * kUnit ? launch<256>(*a, ranks, s) : launch<512>(*a, ranks, s);
}
