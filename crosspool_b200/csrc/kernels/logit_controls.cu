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

#include <atomic>
#include <utility>

#include "xpool/elem.cuh"
#include "xpool/gumbel.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace controls {

constexpr int kSlots = 4096;                       // tokens of a share that can be counted at once
constexpr int kSearch = 64;                        // slots that a token is searched in; one that finds no room is counted in another round
constexpr uint32_t kEmpty = 0xffffffffu;
constexpr uint32_t kInPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;
constexpr int kMaxRanks = 8;
constexpr int kBatch = 4;                          // loads of a thread in flight (kSlots is a multiple of 1024 * kBatch)
constexpr int kUnit = 1024;                        // shares are multiples of so many tokens

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

// (loads that do not hang on one another stand side by side: a chain of them is a microsecond of a small batch)
__device__ __forceinline__ Row load_row(const XpLogitArgs& a, int r) {
  const XpLogitControls& c = a.c;
  Row w;
  const int slot = c.history_rows != nullptr ? c.history_rows[r] : r;
  const int len = c.history != nullptr ? c.lens[r] : 0;
  const int prompt = c.prompt_lens != nullptr ? c.prompt_lens[r] : 0;
  const int latest = c.latest != nullptr ? c.latest[r] : -1;
  const int bias0 = c.bias_starts != nullptr ? c.bias_starts[r] : 0, bias1 = c.bias_starts != nullptr ? c.bias_starts[r + 1] : 0;
  const int m = c.mask_index != nullptr ? c.mask_index[r] : -1;
  const float t = a.temps != nullptr ? a.temps[r] : 0.f;
  w.repetition = c.repetition != nullptr ? c.repetition[r] : 1.f;
  w.frequency = c.frequency != nullptr ? c.frequency[r] : 0.f;
  w.presence = c.presence != nullptr ? c.presence[r] : 0.f;
  const bool known = slot >= 0 && slot < c.history_slots;
  w.history = known ? c.history + static_cast<size_t>(slot) * c.ld_history : nullptr;
  w.len = known ? min(max(len, 0), c.history_cap) : 0;
  w.prompt = prompt;
  w.latest = w.len > 0 ? latest : -1;
  w.bias0 = min(max(bias0, 0), c.bias_total);
  w.bias1 = min(max(bias1, w.bias0), c.bias_total);
  w.mask = m >= 0 && m < c.mask_count ? c.masks + static_cast<size_t>(m) * c.ld_mask : nullptr;
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

// The largest of those of 16 bytes of logits whose bits are set (-inf if none is).
__device__ __forceinline__ float largest(const uint4& v, uint32_t use, float) {
  const float low = -CUDART_INF_F;
  const float x = use & 1u ? __uint_as_float(v.x) : low, y = use & 2u ? __uint_as_float(v.y) : low;
  const float z = use & 4u ? __uint_as_float(v.z) : low, w = use & 8u ? __uint_as_float(v.w) : low;
  return fmaxf(fmaxf(x, y), fmaxf(z, w));
}
// (bf16: four bits become the signs of four bytes, and those two pairs of half-word masks)
__device__ __forceinline__ float largest(const uint4& v, uint32_t use, __nv_bfloat16) {
  uint32_t r[4] = {v.x, v.y, v.z, v.w};
  if (use != 0xffu) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t signs = (((use >> (4 * h)) & 15u) * 0x00204081u & 0x01010101u) << 7;
      uint32_t m0, m1;                               // (the intrinsic leaves out the mode that spreads a byte's sign)
      asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m0) : "r"(signs));
      asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m1) : "r"(signs));
      r[2 * h] = (r[2 * h] & m0) | (0xff80ff80u & ~m0);
      r[2 * h + 1] = (r[2 * h + 1] & m1) | (0xff80ff80u & ~m1);
    }
  }
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(r);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Occurrences of marked tokens, found by linear search from a hashed place: the factor is odd, so kSlots neighbouring tokens have
// places of their own.
struct Table {
  uint32_t* keys;
  uint32_t* words;
  __device__ __forceinline__ static int place(uint32_t id) { return static_cast<int>((id * 2654435761u) & (kSlots - 1)); }
  // the slot of a token, which is entered where it is not there; -1: no room
  __device__ __forceinline__ int enter(uint32_t id) const {
    int s = place(id);
    for (int i = 0; i < kSearch; ++i, s = (s + 1) & (kSlots - 1)) {
      const uint32_t k = atomicCAS(&keys[s], kEmpty, id);
      if (k == kEmpty || k == id) return s;
    }
    return -1;
  }
  __device__ __forceinline__ uint32_t word(uint32_t id) const {
    for (int s = place(id);; s = (s + 1) & (kSlots - 1))
      if (keys[s] == id) return words[s];
  }
};

// kOdd: rows whose pitch is no whole 16 bytes (their vectors' bits in masks and marks begin anywhere in a word).
template <typename T, typename O, bool kSelect, bool kOdd, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
logit_controls_kernel(XpLogitArgs a, int wide, int ranks, int share) {
  namespace cg = cooperative_groups;
  constexpr int N = 16 / sizeof(T), kWarps = kThreads / 32;
  __shared__ float keys_s[kMaxRanks * kWarps], vals_s[kMaxRanks * kWarps];
  __shared__ int toks_s[kMaxRanks * kWarps];
  __shared__ int repeats;
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
    if (w.noisy) k -= gumbel::minus_noise(w.seed, w.step, static_cast<uint32_t>(i));
    return k;
  };

  // The next loads of a thread are always in flight: while marks are made, and while loaded logits are worked on.
  // Rows of an odd vocabulary begin anywhere: vectors begin behind the `head` tokens before the first whole 16 bytes.
  const int head = kOdd ? min(n, static_cast<int>((N - static_cast<size_t>(r) * a.ld % N) % N)) : 0, whole = wide ? (n - head) / N : 0, lov = lo + head;
  uint4 ahead[kBatch];
  // ... the mask's bits of the same tokens: a byte, or the two words that they lie in; shifted when they are used, or the loads
  // would be waited for here
  uint32_t bits[kBatch], more[kOdd ? kBatch : 1];
  auto bits_at = [](const uint32_t* p, int at, int last) {     // 32 bits from a place on; `last`: the last word that is there
    return __funnelshift_r(p[at >> 5], p[min((at >> 5) + 1, last)], at & 31);
  };
  auto fetch = [&](int c) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (c + j * kThreads < whole) {
        ahead[j] = reinterpret_cast<const uint4*>(row + lov)[c + j * kThreads];
        const int i0 = lov + (c + j * kThreads) * N;
        bits[j] = ~0u;
        if constexpr (kOdd) {
          more[j] = ~0u;
          if (w.mask != nullptr) bits[j] = w.mask[i0 >> 5], more[j] = w.mask[min((i0 >> 5) + 1, (a.vocab - 1) >> 5)];
        } else {
          if (w.mask != nullptr) bits[j] = reinterpret_cast<const uint8_t*>(w.mask)[i0 >> 3];
        }
      }
  };
  fetch(threadIdx.x);

  // ---- marks and counts of the tokens that the controls touch
  // tokens [t0, t1): returns whether they found room
  auto count = [&](int t0, int t1, bool mark) {
    int ids[kBatch];
    auto get = [&](int i0) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads;
        ids[j] = i < w.len ? w.token(i) : -1;
      }
    };
    get(threadIdx.x);
    if (threadIdx.x == 0) repeats = 0;
    for (int i = threadIdx.x * 4; i < kSlots; i += kThreads * 4) {
      *reinterpret_cast<uint4*>(table.keys + i) = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
      *reinterpret_cast<uint4*>(table.words + i) = make_uint4(0, 0, 0, 0);
    }
    if (mark)
      for (int i = threadIdx.x * 4; i < (n + 31) / 32; i += kThreads * 4) *reinterpret_cast<uint4*>(marks + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    bool full = false;
    auto enter = [&](int id, uint32_t what) -> uint32_t {
      if (mark) atomicOr(&marks[(id - lo) >> 5], 1u << ((id - lo) & 31));
      const int s = full ? -1 : table.enter(static_cast<uint32_t>(id));
      if (s < 0) {
        full = true;
        return 0u;
      }
      return what == 1u ? atomicAdd(&table.words[s], 1u) : atomicOr(&table.words[s], what);
    };
    for (int i = threadIdx.x; i < w.len; i += kThreads * kBatch) {
      int now[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) now[j] = ids[j];
      if (i + kThreads * kBatch < w.len) get(i + kThreads * kBatch);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (now[j] >= t0 && now[j] < t1) enter(now[j], i + j * kThreads < w.prompt ? kInPrompt : 1u);
    }
    for (int e = w.bias0 + threadIdx.x; e < w.bias1; e += kThreads) {
      const int id = a.c.bias_ids[e];
      if (id >= t0 && id < t1 && (enter(id, kBiased) & kBiased)) repeats = 1;
    }
    return __syncthreads_or(full) == 0;
  };
  const bool fits = !touched || count(lo, hi, true);

  // ---- the stream: tokens without marks
  int at = -1;                                     // first token of the vector that holds the best one
  auto stream = [&](int i0, const uint4& raw, uint32_t allowed) {
    const T* v = reinterpret_cast<const T*>(&raw);
    constexpr uint32_t ones = (1u << N) - 1u;
    const uint32_t skip = !touched ? 0u : !kOdd ? marks[(i0 - lo) >> 5] >> ((i0 - lo) & 31) & ones : bits_at(marks, i0 - lo, (n - 1) >> 5) & ones;
    const uint32_t use = allowed & ~skip & ones;
    if constexpr (kSelect) {
      if (w.noisy) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float f = allowed >> j & 1u ? as_float(v[j]) : -CUDART_INF_F;
          if (!(skip >> j & 1u)) best.offer(key_of(f, i0 + j), f, i0 + j);
        }
        return;
      }
      // only the value and the vector's place; which of its tokens it is, is looked up once, at the end
      const float top = largest(raw, use, T());
      at = top > best.key || at < 0 ? i0 : at;
      best.key = fmaxf(best.key, top);
    } else {
      O* to = out + i0;
      if (sizeof(O) == sizeof(T) && (allowed & ones) == ones) {
        *reinterpret_cast<uint4*>(to) = raw;
        return;
      }
      __align__(16) O o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) elem::st(o + j, (allowed | skip) >> j & 1u ? as_float(v[j]) : -CUDART_INF_F);   // marked tokens stay as they are for now
      if constexpr (sizeof(O) * N == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(o);
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(O)) * N / 16; ++j) reinterpret_cast<uint4*>(to)[j] = reinterpret_cast<const uint4*>(o)[j];
    }
  };
  for (int c = threadIdx.x; c < whole; c += kThreads * kBatch) {
    uint4 now[kBatch];
    uint32_t allowed[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i0 = lov + (c + j * kThreads) * N;
      now[j] = ahead[j];
      allowed[j] = kOdd ? __funnelshift_r(bits[j], more[kOdd ? j : 0], i0 & 31) : bits[j] >> (i0 & 7);
    }
    fetch(c + kThreads * kBatch);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (c + j * kThreads < whole) stream(lov + (c + j * kThreads) * N, now[j], allowed[j]);
  }
  if constexpr (kSelect) {
    if (at >= 0 && !w.noisy) {
      const uint4 raw = *reinterpret_cast<const uint4*>(row + at);
      const T* v = reinterpret_cast<const T*>(&raw);
      const uint32_t skip = touched ? bits_at(marks, at - lo, (n - 1) >> 5) : 0u, allowed = w.mask != nullptr ? bits_at(w.mask, at, (a.vocab - 1) >> 5) : ~0u;
      best.value = best.key;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        const float f = allowed >> j & 1u ? as_float(v[j]) : -CUDART_INF_F;
        if (!(skip >> j & 1u) && f == best.key) best.token = at + j;
      }
    }
  }
  for (int k = threadIdx.x; k < n - whole * N; k += kThreads) {      // before and behind them
    const int i = k < head ? lo + k : lo + whole * N + k;
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
#pragma unroll 1
    for (int s0 = threadIdx.x; s0 < kSlots; s0 += kThreads * kBatch) {
      uint32_t id[kBatch];
      T raw[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        id[j] = table.keys[s0 + j * kThreads];
        if (id[j] != kEmpty) raw[j] = row[id[j]];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint32_t word = table.words[s0 + j * kThreads];
        if (id[j] != kEmpty && !(word & kBiased)) finish(static_cast<int>(id[j]), penalised(as_float(raw[j]), word, w));
      }
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
      // more tokens than the table holds: as many neighbouring ones as there are slots, one range after the other
      for (int t0 = lo; t0 < hi; t0 += kSlots) {
        const int t1 = min(t0 + kSlots, hi);
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
      a.tokens[r] = b.token == 0x7fffffff ? 0 : b.token;       // nothing but NaN
      if (a.values != nullptr) a.values[r] = b.value;
    }
  }
}

template <auto kernel, int kThreads>
static int go(const XpLogitArgs& a, int wide, int ranks, int share, int smem, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};           // devices on which the kernel may have the shared memory
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

template <bool kOdd, int kThreads>
static int launch_as(const XpLogitArgs& a, int wide, int ranks, int share, int smem, cudaStream_t s) {
  using bf16 = __nv_bfloat16;
  if (a.out == nullptr) return a.f32 ? go<logit_controls_kernel<float, float, true, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
                                     : go<logit_controls_kernel<bf16, float, true, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
  if (a.out_f32) return a.f32 ? go<logit_controls_kernel<float, float, false, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
                              : go<logit_controls_kernel<bf16, float, false, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
  return a.f32 ? go<logit_controls_kernel<float, bf16, false, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s)
               : go<logit_controls_kernel<bf16, bf16, false, kOdd, kThreads>, kThreads>(a, wide, ranks, share, smem, s);
}

template <int kThreads>
static int launch(const XpLogitArgs& a, int ranks, cudaStream_t s) {
  const int es = a.f32 ? 4 : 2, eo = a.out == nullptr ? 16 : a.out_f32 ? 4 : 2;
  auto based = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool whole = a.ld * es % 16 == 0 && (a.out == nullptr || a.ld_out * eo % 16 == 0);
  // 16 bytes a load where logits and result are aligned alike in every row
  const int wide = based(a.logits) && based(a.out) && (whole || a.out == nullptr || a.ld == a.ld_out);
  const int share = ((a.vocab + ranks - 1) / ranks + kUnit - 1) / kUnit * kUnit;
  const int smem = 2 * kSlots * 4 + share / 8;
  return wide && !whole ? launch_as<true, kThreads>(a, wide, ranks, share, smem, s) : launch_as<false, kThreads>(a, wide, ranks, share, smem, s);
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
  // About 256 CTAs of 512 threads, of which an SM holds two. us, CTAs a row 1 / 2 / 4 / 8: 256 rows of 151936 with histories and masks
  // 33 / 39 / 55 / 86, 64 rows 22 / 16 / 16 / 24, 16 rows 20 / 14 / 11 / 11, 3 rows 17 / 12 / 9 / 8.
  int ranks = a->rows <= 32 ? 8 : a->rows <= 64 ? 4 : a->rows <= 128 ? 2 : 1;
  while (ranks > 1 && a->vocab / ranks < 4 * kUnit) ranks >>= 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->vocab / ranks <= 4 * kUnit ? launch<256>(*a, ranks, s) : launch<512>(*a, ranks, s);
}
