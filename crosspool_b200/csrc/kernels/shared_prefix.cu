// Decode attention of rows that share prefixes: the prefix of a group of rows is multiplied once for all of them on the Blackwell
// tensor cores, while other warps of the same CTAs stream the tokens of each row's own. Both leave partial results, un-normalised
// sums O = sum_t 2^(s_t - m) v_t with their maximum m and sum of weights l; a second kernel merges them.
//
// The two kinds of work are bound by different things: M rows on a prefix of n tokens are 4 M G n d operations for 4 n d bytes
// (tensor pipe and exponentials), own tokens are one read of the cache. One kernel after the other, 256 rows of four heads on 8192
// tokens with 165 tokens of their own took 45 + 54 us. So a persistent grid does both at once, some SMs the one and some the other:
//
// Pieces. A plan cuts every prefix into pieces (a range of its tokens, and up to 2 x (128 / G) consecutive rows that read it, G
// query heads to a KV head). The first CTAs take (piece, KV head) units in turn: two tiles of 128 queries (row of a tile = row * G
// + head), both multiplied against the same steps of 128 tokens, so that the tensor pipe works on one while the softmax of the other runs.
//   warps 0-3   softmax of tile A: thread = query = TMEM lane. Reads its row of S with tcgen05.ld, keeps a running maximum and
//               sum, writes P (bf16) over the second half of S as the A operand of the second product, rescales O in tensor memory only
//               when the maximum grew by more than 2^8 (sum and result carry the same stale maximum), and stores the partial result.
//   warps 4-7   the same for tile B.
//   warp 8      TMA producer: Q tiles once a unit, then a ring of steps of keys and values through the leader's page table (128-byte swizzle).
//   warp 9      allocates tensor memory and issues every tcgen05.mma: PV_A(t), S_A(t+1), PV_B(t), S_B(t+1).
// Own tokens. The 16-token tiles of all rows' own tokens, row by row, KV head by KV head, are one list that is cut into shares for
// the warps of the grid, wherever a share ends: ragged rows balance, and a row's tokens are in at most own_slots shares. CTAs
// without pieces begin at once and get larger shares, by as much as the others' pieces take.
//   warps 0-11  a worker each, with a ring of its own filled by TMA (an SM keeps up to 192 KB in flight: half of them carry the
//               whole bandwidth). Products transposed, S^T = K Q^T and O^T = V^T P^T by mma.m16n8k16: tokens (then head dims) fill
//               the 16 rows, the up to 8 query heads of a unit the 8 columns, so nothing is padded; P^T becomes the B operand by
//               two 8 x 8 transposes. (9 to 16 heads are two units.)
//
// P is rounded to bf16 for the second product (2^-8 of a weight at most, as in prefill attention); l sums the unrounded weights.
// The last tile of a prefix or of a row may end inside: scores behind the end are selected away and the values zeroed, whatever
// the cache holds there. Every wait is bounded; one that runs out sets the abort word, the status word (13) and ends the CTA
// behind a common barrier.
#include <math_constants.h>

#include <atomic>

#include "xpool/mma_sync.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"
#include "xpool/sm100.cuh"
#include "xpool/tensormap.hpp"

namespace xpool {
namespace prefix {

constexpr int kRows = 128;       // queries of a tile (UMMA M)
// Tokens of a step. Scores in products of 128 columns take as long as in products of 64 (counters: the tensor pipe was busy for
// 1600 cycles per 64 tokens and two query tiles instead of 1024).
constexpr int kBN = 128;
constexpr int kStages = 2;
constexpr int kWarps = 12;
constexpr int kThreads = 32 * kWarps;
constexpr float kRescaleStep = 8.0f;   // log2 units
constexpr uint32_t kMinShare = 2;      // tiles of a worker's share, at least
// Time of a unit of pieces, in tiles of own tokens that a CTA streams meanwhile: once, and for each of its steps.
constexpr uint32_t kUnitCost = 35, kTileCost = 19;
template <int D>
constexpr int ring_of() { return 256 / D; }   // tiles of a worker's ring: 16 KB

struct __align__(8) Bars {
  uint64_t q_full, q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages];
  uint64_t v_full[kStages], v_empty[kStages];
  uint64_t s_full[2];
  uint64_t p_half[2], p_full[2];
  uint64_t pv_done[2];
  uint64_t own_full[kWarps][4];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
  uint32_t own_sum[2], own_max[2];
};

// Where the partial results of head hq of row b lie.
struct Partials {
  float* sums;
  float2* pairs;
  __device__ __forceinline__ Partials(const XpDecodeSharedArgs& s, int D, int b, int hq) {
    const int slots = s.max_parts + s.own_slots;
    const size_t all = static_cast<size_t>(s.a.batch) * s.a.q_heads * slots, at = (static_cast<size_t>(b) * s.a.q_heads + hq) * slots;
    sums = s.a.ws + at * D;
    pairs = reinterpret_cast<float2*>(s.a.ws + all * D) + at;
  }
};
// Behind them: the shares, and the first tile of every row, in units of one KV head's tiles (written by the last CTA).
__device__ __forceinline__ uint32_t* share_words(const XpDecodeSharedArgs& s, int D) {
  return reinterpret_cast<uint32_t*>(s.a.ws + static_cast<size_t>(s.a.batch) * s.a.q_heads * (s.max_parts + s.own_slots) * (D + 2));
}
// Workers [0, free) take `large` tiles each, those behind them `small` (none where that is 0).
struct Shares {
  uint32_t free, large, small;
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w < free ? w * large : free * large + (w - free) * small; }
  __device__ __forceinline__ uint32_t size(uint32_t w) const { return w < free ? large : small; }
  __device__ __forceinline__ uint32_t worker(uint32_t tile) const { return tile < free * large ? tile / large : free + (tile - free * large) / small; }
};
__device__ __forceinline__ int row_tokens(const XpDecodeSharedArgs& s, int b) { return min(max(s.a.seq_lens[b], 0), s.max_len); }
// Tokens that row b shares: none where it has fewer than the prefix.
__device__ __forceinline__ int shared_tokens(const XpDecodeSharedArgs& s, int b) {
  const int p = b < s.plan_rows ? s.row_prefix[b] : 0;
  return row_tokens(s, b) >= p ? p : 0;
}
// Units that a row's tokens are multiplied in: KV heads, twice where 9 to 16 query heads share one.
__device__ __forceinline__ int row_units(const XpDecodeAttnArgs& a) { return a.q_heads / a.kv_heads > 8 ? 2 * a.kv_heads : a.kv_heads; }

// Bounded wait of a converged warp that also gives up when another role of the CTA has; one answer for all lanes.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* b, uint32_t site) {
  bool ok = false;
  uint64_t deadline = 0;                            // the timer is read only once a wait has become a long one
  for (uint32_t spins = 1; !(ok = sm100::mbar_try_wait(bar, parity)); ++spins) {
    if ((spins & 0xffu) != 0) continue;
    if (b->abort_flag != 0) break;
    const uint64_t now = sm100::global_timer_ns();
    if (deadline == 0) deadline = now + sm100::kPipelineWaitNs;
    if (now > deadline) {
      b->abort_flag = site;
      break;
    }
  }
  return __all_sync(0xffffffffu, ok) != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Two weights (not negative) rounded to bf16, ties up. The conversion instruction runs on the unit of the exponentials, an eighth of
// a warp a cycle, and made it half as busy again; additions and a byte permutation do not. (NaN may be lost here; the sum keeps it.)
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  return __byte_perm(__float_as_uint(lo) + 0x8000u, __float_as_uint(hi) + 0x8000u, 0x7632);
}
// Two fp32 numbers in one register pair, computed by one instruction.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float2 parts_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// For every row its first tile (first[batch]: their number), and the tokens it shares | the tokens of its last tile - 1. bars.own_max:
// the most tiles of a row. Two warps, which have no part in the pieces.
constexpr int kScanThreads = 64;
__device__ __forceinline__ void scan_rows(const XpDecodeSharedArgs& args, Bars& bars, uint32_t* first, uint32_t* place, int tid) {
  const int batch = args.a.batch, lane = tid & 31, each = (batch + kScanThreads - 1) / kScanThreads;
  const int b0 = min(batch, tid * each), b1 = min(batch, b0 + each);
  uint32_t sum = 0, most = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const int shared = shared_tokens(args, b), own = row_tokens(args, b) - shared;
    const uint32_t n = static_cast<uint32_t>(own + 15) >> 4;
    first[b] = n, place[b] = static_cast<uint32_t>(shared) | ((own - 1) & 15);
    sum += n, most = max(most, n);
  }
  uint32_t before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (lane == 31) bars.own_sum[tid >> 5] = before;
  if (lane == 0) bars.own_max[tid >> 5] = most;
  asm volatile("bar.sync 1, %0;" ::"n"(kScanThreads) : "memory");
  uint32_t at = before - sum + (tid >= 32 ? bars.own_sum[0] : 0u);
  for (int b = b0; b < b1; ++b) {
    const uint32_t n = first[b];
    first[b] = at;
    at += n;
  }
  if (tid == kScanThreads - 1) first[batch] = at;
}

// Shares of `total` tiles for `busy` CTAs that have spent the time of `cost` tiles on pieces and `idle` CTAs that have not.
__device__ __forceinline__ Shares make_shares(uint32_t total, uint32_t most, int own_slots, uint32_t busy, uint32_t idle, uint32_t cost) {
  const uint32_t least = max(kMinShare, (most + own_slots - 2) / (own_slots - 1));     // a row is in at most own_slots shares
  uint32_t mine = 0, theirs = 0;                                                      // tiles of an idle CTA, of a busy one
  if (idle > 0 && total <= static_cast<unsigned long long>(idle) * cost) {
    mine = (total + idle - 1) / idle;
  } else {
    theirs = total > idle * cost ? (total - idle * cost + busy + idle - 1) / (busy + idle) : 0;
    mine = theirs + cost;
  }
  Shares s;
  s.free = idle * kWarps;
  s.large = max(least, (mine + kWarps - 1) / kWarps);
  s.small = theirs > 0 ? max(least, (theirs + kWarps - 1) / kWarps) : 0;
  if (s.free * static_cast<unsigned long long>(s.large) >= total) s.small = 0;
  return s;
}

// Lane i's tile of a block of 32 tiles of a share: its row, unit, place in the row's own tokens, and place in the cache.
struct Tile {
  int row, unit, tile, own, tok;
};

template <int D>
__device__ __forceinline__ void own_worker(const CUtensorMap* tmap_k, const CUtensorMap* tmap_v, const XpDecodeSharedArgs& args, Bars& bars,
                                           const uint32_t* first, const uint32_t* place, const Shares shares, uint32_t number, uint32_t ring, int w,
                                           int lane, int G) {
  const XpDecodeAttnArgs& a = args.a;
  constexpr int kRing = ring_of<D>(), kHalves = D / 64, kBox = 16 * 128, kTile = 2 * kHalves * kBox;    // K boxes of 16 tokens x 64 dims, then V boxes
  const uint32_t units = row_units(a), total = first[a.batch] * units, mine = shares.begin(number);
  if (mine >= total) return;
  const int n = static_cast<int>(min(shares.size(number), total - mine));

  const int page_shift = 31 - __clz(a.page_size), page_mask = a.page_size - 1;
  auto look = [&](int block) {
    Tile t{0, 0, 0, 0, 0};
    const int i = block * 32 + lane;
    if (i >= n) return t;
    const uint32_t j = mine + i, x = j / units;
    int lo = 0, hi = a.batch;                       // first[lo] <= x < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= x) lo = mid;
      else hi = mid;
    }
    const uint32_t tiles = first[lo + 1] - first[lo], at = j - first[lo] * units, skip = place[lo] & ~15u;
    t.row = lo, t.unit = at / tiles, t.tile = at - t.unit * tiles;
    t.own = static_cast<int>((tiles - 1) * 16 + (place[lo] & 15u) + 1);
    const int ts = static_cast<int>(skip) + t.tile * 16;
    t.tok = (a.block_table[static_cast<size_t>(lo) * a.max_blocks + (ts >> page_shift)] << page_shift) + (ts & page_mask);
    return t;
  };
  const int per = units == a.kv_heads ? 1 : 2;      // units of a KV head
  Tile now = look(0), next = n > 32 ? look(1) : now;
  auto issue = [&](int i, const Tile& t) {
    const int tok = __shfl_sync(0xffffffffu, t.tok, i & 31), hk = __shfl_sync(0xffffffffu, t.unit, i & 31) / per;
    uint64_t* full = &bars.own_full[w][i % kRing];
    if (lane == 0) {
      sm100::mbar_arrive_expect_tx(full, kTile);
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        sm100::tma_load_3d_addr(ring + (i % kRing) * kTile + h * kBox, tmap_k, sm100::smem_u32(full), h * 64, hk, tok);
        sm100::tma_load_3d_addr(ring + (i % kRing) * kTile + (kHalves + h) * kBox, tmap_v, sm100::smem_u32(full), h * 64, hk, tok);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i)
    if (i < n) issue(i, now);

  const int g = lane >> 2, q4 = lane & 3;
  const float sc2 = a.scale * 1.4426950408889634f;
  uint32_t qf[D / 16][2];                           // Q^T: head g, dims 16 ks + 2 q4 .. (+ 8)
  float acc[D / 16][4];                             // O^T: dims 16 j + g (+ 8), heads 2 q4, 2 q4 + 1
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
  const int a_row = lane & 15, a_chunk = lane >> 4;                               // ldmatrix rows of K (16 tokens x 16 dims)
  const int t_row = (lane & 7) + (lane >> 4) * 8, t_chunk = (lane >> 3) & 1;      // ... of V, transposed
  for (int i = 0; i < n; ++i) {
    const int src = i & 31;
    const int row = __shfl_sync(0xffffffffu, now.row, src), unit = __shfl_sync(0xffffffffu, now.unit, src);
    const int tile = __shfl_sync(0xffffffffu, now.tile, src), own = __shfl_sync(0xffffffffu, now.own, src);
    const int heads0 = unit / per * G + unit % per * 8, heads = min(8, G - unit % per * 8);
    if (i == 0 || tile == 0) {
      const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (static_cast<size_t>(row) * a.q_heads + heads0 + g) * D + q4 * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][0] = g < heads ? *reinterpret_cast<const uint32_t*>(q + ks * 16) : 0u;
        qf[ks][1] = g < heads ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 8) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[ks][e] = 0.f;
      }
      m0 = m1 = -CUDART_INF_F, l0 = l1 = 0.f;
    }
    if (!wait_bar(&bars.own_full[w][i % kRing], (i / kRing) & 1, &bars, 11)) return;
    const uint32_t st = ring + (i % kRing) * kTile;
    const int nvalid = own - tile * 16;
    if (nvalid < 16) {
      // cache slots behind the sequence's end may hold anything: zero those V rows (a weight of zero times NaN)
      for (int z = lane; z < (16 - nvalid) * kHalves * 8; z += 32) {
        const int r = nvalid + z / (kHalves * 8), rest = z % (kHalves * 8);
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(st + (kHalves + rest / 8) * kBox + r * 128 + (rest % 8) * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};     // tokens g (+ 8), heads 2 q4, 2 q4 + 1; two chains of products
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int cc = 2 * ks + a_chunk;
      uint32_t kf[4];
      frag::ldsm4(st + (cc >> 3) * kBox + a_row * 128 + (((cc & 7) ^ (a_row & 7)) << 4), kf);
      frag::mma(s[ks & 1], kf, qf[ks][0], qf[ks][1]);
    }
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = g + (e >> 1) * 8 < nvalid ? (s[0][e] + s[1][e]) * sc2 : -CUDART_INF_F;
    float x0 = fmaxf(v[0], v[2]), x1 = fmaxf(v[1], v[3]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
    }
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
      const float c0 = n0 > m0 ? exp2f(m0 - n0) : 1.f, c1 = n1 > m1 ? exp2f(m1 - n1) : 1.f;
      l0 *= c0, l1 *= c1, m0 = n0, m1 = n1;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) acc[j][0] *= c0, acc[j][1] *= c1, acc[j][2] *= c0, acc[j][3] *= c1;
    }
    // (keys that hold an infinity may leave no score above -inf so far: weights of 0 then)
    const float z0 = m0 == -CUDART_INF_F ? 0.f : m0, z1 = m1 == -CUDART_INF_F ? 0.f : m1;
    const float p0 = exp2f(v[0] - z0), p1 = exp2f(v[1] - z1), p2 = exp2f(v[2] - z0), p3 = exp2f(v[3] - z1);
    l0 += p0 + p2, l1 += p1 + p3;
    const uint32_t b0 = transpose8x8(pack2(p0, p1)), b1 = transpose8x8(pack2(p2, p3));
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const int cc = 2 * j + t_chunk;
      uint32_t vf[4];
      frag::ldsm4t(st + (kHalves + (cc >> 3)) * kBox + t_row * 128 + (((cc & 7) ^ (t_row & 7)) << 4), vf);
      frag::mma(acc[j], vf, b0, b1);
    }
    __syncwarp();                                    // every lane has consumed the tile
    if (i + kRing < n) {
      sm100::fence_proxy_async_smem();
      issue(i + kRing, (i + kRing) >> 5 == i >> 5 ? now : next);
    }
    if (i == n - 1 || (tile + 1) * 16 >= own) {      // the unit's last tile of this share
      float a0 = l0, a1 = l1;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) a0 += __shfl_xor_sync(0xffffffffu, a0, o), a1 += __shfl_xor_sync(0xffffffffu, a1, o);
      const uint32_t start = first[row] * units + static_cast<uint32_t>(unit) * (first[row + 1] - first[row]);
      const int slot = args.max_parts + static_cast<int>(number - shares.worker(start));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * q4 + h >= heads) continue;
        const Partials p(args, D, row, heads0 + 2 * q4 + h);
        float* o = p.sums + static_cast<size_t>(slot) * D + g;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[16 * j] = acc[j][h], o[16 * j + 8] = acc[j][2 + h];
        if (g == 0) p.pairs[slot] = make_float2(h ? m1 : m0, h ? a1 : a0);
      }
    }
    if (src == 31 && i + 1 < n) now = next, next = look((i >> 5) + 2);
  }
}

__device__ __forceinline__ void tmem_ld_wait16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const __grid_constant__ CUtensorMap tmap_k16, const __grid_constant__ CUtensorMap tmap_v16,
                     const __grid_constant__ XpDecodeSharedArgs args, int G, int box_tokens) {
  constexpr int kHalves = D / 64;                 // 64-dim (128-byte) column blocks of a row
  constexpr int kQHalf = kRows * 128;
  constexpr int kQTile = kHalves * kQHalf;
  constexpr int kKVHalf = kBN * 128;
  constexpr int kKTile = kHalves * kKVHalf;
  constexpr int kStage = 2 * kKTile;              // K then V
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kOCol = 2 * kBN;             // S_A, S_B (P over the second half of either), then O_A, O_B
  constexpr uint32_t kPCol = kBN / 2;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ Bars bars;

  pdl::wait();
  const XpDecodeAttnArgs& a = args.a;
  const int n_units = min(*args.n_pieces, args.max_pieces) * a.kv_heads;
  const int np = kRows / G;                       // rows of a tile; its last 128 - np G queries are none
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (sm100::smem_u32(smem_dyn) + 1023u) & ~1023u;
  const uint32_t q_s = base, kv_s = base + 2 * kQTile;
  constexpr int kTiles = 2 * kQTile + kStages * kStage, kRings = kWarps * ring_of<D>() * 16 * D * 4;
  uint32_t* first = reinterpret_cast<uint32_t*>(smem_dyn + (base - sm100::smem_u32(smem_dyn)) + (kTiles > kRings ? kTiles : kRings));
  uint32_t* place = first + XP_PREFIX_ROWS + 1;
  // the first `busy` CTAs take the units of pieces, `turns` of them each
  const int turns = (n_units + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), busy = turns > 0 ? (n_units + turns - 1) / turns : 0;
  const bool has_units = static_cast<int>(blockIdx.x) < busy;

  if (threadIdx.x == 32) {
    sm100::tma_prefetch_desc(&tmap_k16);
    sm100::tma_prefetch_desc(&tmap_v16);
    sm100::tma_prefetch_desc(&tmap_q);
    sm100::tma_prefetch_desc(&tmap_k);
    sm100::tma_prefetch_desc(&tmap_v);
  }
  if (threadIdx.x == 0) {
    sm100::mbar_init(&bars.q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      sm100::mbar_init(&bars.k_full[s], 1);
      sm100::mbar_init(&bars.k_empty[s], 1);
      sm100::mbar_init(&bars.v_full[s], 1);
      sm100::mbar_init(&bars.v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      sm100::mbar_init(&bars.q_empty[x], 4);
      sm100::mbar_init(&bars.s_full[x], 1);
      sm100::mbar_init(&bars.p_half[x], 4);
      sm100::mbar_init(&bars.p_full[x], 4);
      sm100::mbar_init(&bars.pv_done[x], 1);
    }
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < 4; ++i) sm100::mbar_init(&bars.own_full[w][i], 1);
    bars.abort_flag = 0;
    sm100::mbar_fence_init();
    sm100::fence_proxy_async_smem();
  }
  if (warp == 9 && has_units) {
    sm100::tmem_alloc(&bars.tmem_base, kTmemCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  const uint32_t tmem = bars.tmem_base;
  pdl::release();

  if (warp > 9) {
    scan_rows(args, bars, first, place, threadIdx.x - 320);
  } else if (!has_units) {
    // nothing before the own tokens
  } else if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    const int page_shift = 31 - __clz(a.page_size), page_mask = a.page_size - 1;
    const int copies = kHalves * (kBN / box_tokens);
    const uint32_t q_bytes = static_cast<uint32_t>(2 * kHalves * np * G * 128);
    int it = 0, ord = 0, both = 0;                // stages; units; units of two query tiles
    bool ok = true, two = false;
    for (int u = blockIdx.x; ok && u < n_units; u += busy, ++ord) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int hk = u % a.kv_heads;
      const int* table = a.block_table + static_cast<size_t>(p.leader) * a.max_blocks;
      if (ord > 0 && !wait_bar(&bars.q_empty[0], (ord - 1) & 1, &bars, 1)) break;
      if (two && !wait_bar(&bars.q_empty[1], (both - 1) & 1, &bars, 1)) break;
      two = p.rows > np, both += two;
      if (lane == 0) sm100::mbar_arrive_expect_tx(&bars.q_full, q_bytes);
      __syncwarp();
      if (lane < 2 * kHalves) {
        const int x = lane / kHalves, h = lane % kHalves;
        sm100::tma_load_3d_addr(q_s + x * kQTile + h * kQHalf, &tmap_q, sm100::smem_u32(&bars.q_full), h * 64, hk * G, p.row0 + x * np);
      }
      const int n_steps = (p.tok1 - p.tok0 + kBN - 1) / kBN;
      for (int t = 0; t < n_steps; ++t, ++it) {
        const int s = it % kStages;
        for (int is_v = 0; ok && is_v < 2; ++is_v) {
          uint64_t* full = is_v ? &bars.v_full[s] : &bars.k_full[s];
          if (it >= kStages && !(ok = wait_bar(is_v ? &bars.v_empty[s] : &bars.k_empty[s], ((it / kStages) - 1) & 1, &bars, 2))) break;
          if (lane == 0) sm100::mbar_arrive_expect_tx(full, kKTile);
          __syncwarp();
          if (lane < copies) {                     // up to 16: blocks of 64 dims, boxes of tokens
            const int h = lane % kHalves, j = lane / kHalves;
            // boxes behind the end repeat the last one
            const int tk = min(p.tok0 + t * kBN + j * box_tokens, (p.tok1 - 1) & ~(box_tokens - 1));
            const int tok = (table[tk >> page_shift] << page_shift) + (tk & page_mask);
            sm100::tma_load_3d_addr(kv_s + s * kStage + is_v * kKTile + h * kKVHalf + j * box_tokens * 128, is_v ? &tmap_v : &tmap_k,
                                    sm100::smem_u32(full), h * 64, hk, tok);
          }
        }
        if (!ok) break;
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer (the whole warp walks, one elected lane issues)
    const bool leader = sm100::elect_one();
    const uint32_t idesc_s = sm100::umma_idesc_bf16(kRows, kBN);
    const uint32_t idesc_o = sm100::umma_idesc_bf16_bmn(kRows, D);
    int it = 0, ord = 0, count[2] = {0, 0};       // stages; units; steps that query tile A (B) has multiplied
    auto issue_s = [&](int x, int i) {            // S_x = Q_x K(i)^T
      if (!leader) return;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t da = sm100::umma_desc_sw128(q_s + x * kQTile + (ks >> 2) * kQHalf) + (ks & 3) * 2;
        const uint64_t db = sm100::umma_desc_sw128(kv_s + (i % kStages) * kStage + (ks >> 2) * kKVHalf) + (ks & 3) * 2;
        sm100::umma_bf16(tmem + static_cast<uint32_t>(x * kBN), da, db, idesc_s, ks > 0 ? 1u : 0u);
      }
      sm100::umma_commit(&bars.s_full[x]);
    };
    auto issue_pv = [&](int x, int i, int half, bool more) {   // O_x (+)= P_x V(i), tokens of one half of the step
      if (!leader) return;
#pragma unroll
      for (int kk = half * (kBN / 32); kk < (half + 1) * (kBN / 32); ++kk) {
        const uint64_t db = sm100::umma_desc_mn_sw128(kv_s + (i % kStages) * kStage + kKTile + kk * 2048, kKVHalf, 1024);
        sm100::umma_bf16_ts(tmem + kOCol + static_cast<uint32_t>(x * D), tmem + static_cast<uint32_t>(x * kBN + kPCol + kk * 8), db, idesc_o,
                            (more || kk > 0) ? 1u : 0u);
      }
      if (half) sm100::umma_commit(&bars.pv_done[x]);
    };
    bool ok = true;
    for (int u = blockIdx.x; ok && u < n_units; u += busy, ++ord) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int n_steps = (p.tok1 - p.tok0 + kBN - 1) / kBN, tiles_x = p.rows > np ? 2 : 1;
      ok = wait_bar(&bars.q_full, ord & 1, &bars, 3) && wait_bar(&bars.k_full[it % kStages], (it / kStages) & 1, &bars, 4);
      if (!ok) break;
      sm100::tc_fence_after_sync();
      for (int x = 0; x < tiles_x; ++x) issue_s(x, it);
      if (leader) sm100::umma_commit(&bars.k_empty[it % kStages]);
      for (int t = 0; ok && t < n_steps; ++t, ++it) {
        for (int x = 0; ok && x < tiles_x; ++x) {
          ok = wait_bar(&bars.p_half[x], count[x] & 1, &bars, 6);
          if (ok && x == 0) ok = wait_bar(&bars.v_full[it % kStages], (it / kStages) & 1, &bars, 12);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          issue_pv(x, it, 0, t > 0);
          ok = wait_bar(&bars.p_full[x], count[x] & 1, &bars, 14);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          issue_pv(x, it, 1, true);
          if (x + 1 == tiles_x && leader) sm100::umma_commit(&bars.v_empty[it % kStages]);
          ++count[x];
          if (t + 1 < n_steps) {
            // the products run in order: the next scores overwrite the weights that the product before them has read
            if (x == 0) ok = wait_bar(&bars.k_full[(it + 1) % kStages], ((it + 1) / kStages) & 1, &bars, 5);
            if (!ok) break;
            sm100::tc_fence_after_sync();
            issue_s(x, it + 1);
            if (x + 1 == tiles_x && leader) sm100::umma_commit(&bars.k_empty[(it + 1) % kStages]);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax and partial results (warps 0-7)
    const int x = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int pos = row / G, head = row % G;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_t = tmem + lane_off + kOCol + static_cast<uint32_t>(x * D);
    const float sc2 = a.scale * 1.4426950408889634f;
    const uint32_t s_t = tmem + lane_off + static_cast<uint32_t>(x * kBN);
    const uint32_t stage = q_s + x * kQTile + (warp & 3) * 4096;   // over the queries of this tile, when they are done with
    int it = 0, c = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < n_units; u += busy) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int n_steps = (p.tok1 - p.tok0 + kBN - 1) / kBN;
      if (x == 0 || p.rows > np) {
        float m_used = -CUDART_INF_F, l = 0.f;
        for (int t = 0; t < n_steps; ++t, ++c) {
          ok = wait_bar(&bars.s_full[x], c & 1, &bars, 7);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          uint32_t lo[kBN / 2], hi[kBN / 2];
          sm100::tmem_ld32_issue(s_t, lo);
          sm100::tmem_ld32_issue(s_t + 32, lo + 32);
          sm100::tmem_ld32_issue(s_t + 64, hi);
          sm100::tmem_ld32_issue(s_t + 96, hi + 32);
          sm100::tmem_ld_wait_all(lo);
          sm100::tmem_ld_wait_all(lo + 32);
          sm100::tmem_ld_wait_all(hi);
          sm100::tmem_ld_wait_all(hi + 32);
          const int nvis = p.tok1 - p.tok0 - t * kBN;       // tokens of the prefix in this step (a uniform number)
          auto cut = [&](uint32_t (&v)[kBN / 2], int n) {
            if (n < kBN / 2) {
#pragma unroll
              for (int j = 0; j < kBN / 2; ++j)
                if (j >= n) v[j] = 0xff800000u;             // -inf: selected, never computed with
            }
          };
          cut(lo, nvis);
          cut(hi, nvis - kBN / 2);
          float mx4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int j = 0; j < kBN / 2; j += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(lo[j + e]), __uint_as_float(hi[j + e]));
          }
          const float m_new = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc2;
          float factor = 1.f;
          if (m_new > m_used + kRescaleStep || m_used == -CUDART_INF_F) {
            if (m_new != -CUDART_INF_F) {
              factor = m_used == -CUDART_INF_F ? 0.f : sm100::ex2_approx(m_used - m_new);
              m_used = m_new;
            }
          }
          const float m_sub = m_used == -CUDART_INF_F ? 0.f : m_used;
          if (t > 0) {
            // the previous second product accumulates into O; it has retired before these scores were complete
            ok = wait_bar(&bars.pv_done[x], (c - 1) & 1, &bars, 8);
            if (!ok) break;
            if (__any_sync(0xffffffffu, factor != 1.f)) {
              sm100::tc_fence_after_sync();
#pragma unroll 1
              for (int e = 0; e < D; e += 16) {
                uint32_t ov[16];
                sm100::tmem_ld16_issue(o_t + e, ov);
                tmem_ld_wait16(ov);
#pragma unroll
                for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * factor);
                tmem_st16(o_t + e, ov);
              }
            }
          }
          if (nvis < kBN && x == 0) {
            // cache slots behind the prefix may hold anything: zero those V rows (a weight of zero times NaN). Tile A's product
            // is issued before tile B's, and both read this stage.
            const uint32_t v_s = kv_s + ((it + t) % kStages) * kStage + kKTile;
            ok = wait_bar(&bars.v_full[(it + t) % kStages], ((it + t) / kStages) & 1, &bars, 13);
            if (!ok) break;
            for (int i = row; i < (kBN - nvis) * (D / 8); i += kRows) {
              const int R = nvis + i / (D / 8), cc = i % (D / 8);
              const uint32_t off = (cc >> 3) * kKVHalf + R * 128 + (((cc & 7) ^ (R & 7)) << 4);
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_s + off), "r"(0u) : "memory");
            }
            sm100::fence_proxy_async_smem();
          }
          // P as the tensor core's A operand: two bf16 to a column, over the second half of S. The second product begins with the
          // step's first half while the weights of the second are computed.
          const uint64_t scale_pair = pair_of(__float_as_uint(sc2), __float_as_uint(sc2));
          const uint64_t off_pair = pair_of(__float_as_uint(-m_sub), __float_as_uint(-m_sub));
          uint64_t sum2[2] = {0, 0};
          auto weights = [&](const uint32_t* v, uint32_t to) {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 e = parts_of(fma2(pair_of(v[j], v[j + 1]), scale_pair, off_pair));
              const float p0 = sm100::ex2_approx(e.x), p1 = sm100::ex2_approx(e.y);
              sum2[(j >> 1) & 1] = add2(sum2[(j >> 1) & 1], pair_of(__float_as_uint(p0), __float_as_uint(p1)));
              pk[j >> 1] = pack_weights(p0, p1);
            }
            tmem_st16(to, pk);
          };
          auto hand_over = [&](uint64_t* bar) {
            sm100::tmem_st_wait();
            sm100::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(bar);
          };
          weights(lo, s_t + kPCol);
          weights(lo + 32, s_t + kPCol + 16);
          hand_over(&bars.p_half[x]);
          weights(hi, s_t + kPCol + 32);
          weights(hi + 32, s_t + kPCol + 48);
          hand_over(&bars.p_full[x]);
          const float2 sum = parts_of(add2(sum2[0], sum2[1]));
          l = l * factor + (sum.x + sum.y);
        }
        if (ok) ok = wait_bar(&bars.pv_done[x], (c - 1) & 1, &bars, 10);
        if (ok) {
          // The partial result goes out through shared memory, 128 bytes of a row at a time: stored from the lanes that hold the
          // rows, 256 rows of 512 bytes kept the store unit for 4 us.
          sm100::tc_fence_after_sync();
          const int r = x * np + pos;
          const bool stored = pos < np && r < p.rows;
          const Partials to(args, D, p.row0 + (stored ? r : 0), min((u % a.kv_heads) * G + head, a.q_heads - 1));
          const unsigned long long mine = stored ? reinterpret_cast<unsigned long long>(to.sums + static_cast<size_t>(p.part) * D) : 0ull;
          if (stored) to.pairs[p.part] = make_float2(m_used, l);
#pragma unroll 1
          for (int e = 0; e < D; e += 32) {
            uint32_t ov[32];
            sm100::tmem_ld32_issue(o_t + e, ov);
            sm100::tmem_ld_wait_all(ov);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(ov[4 * j]), "r"(ov[4 * j + 1]),
                           "r"(ov[4 * j + 2]), "r"(ov[4 * j + 3])
                           : "memory");
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int rr = j * 4 + (lane >> 3), cc = lane & 7;
              const unsigned long long o = __shfl_sync(0xffffffffu, mine, rr);
              uint4 v;
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + rr * 128 + ((cc ^ (rr & 7)) << 4)));
              if (o != 0) reinterpret_cast<uint4*>(o)[e / 4 + cc] = v;
            }
            __syncwarp();
          }
          sm100::tc_fence_before_sync();       // O has been read before the next unit's first arrival at p_full
          sm100::fence_proxy_async_smem();     // the next queries are copied over the staged rows
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&bars.q_empty[x]);
        }
      }
      it += n_steps;
    }
  }
  // ------------------------------------------------------------------ own tokens, over the memory of the pieces' tiles
  sm100::tc_fence_before_sync();
  sm100::fence_proxy_async_smem();
  __syncthreads();
  if (warp == 9 && has_units) {
    sm100::tc_fence_after_sync();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
  const bool failed = bars.abort_flag != 0;         // uniform: every role is behind the barrier
  if (!failed) {
    const uint32_t most = max(bars.own_max[0], bars.own_max[1]);
    const uint32_t idle = gridDim.x - busy, cost = turns * (kUnitCost + kTileCost * ((args.n_pieces[1] + kBN - 1) / kBN));
    const Shares shares = make_shares(first[a.batch] * row_units(a), most, args.own_slots, busy, idle, cost);
    if (blockIdx.x == gridDim.x - 1) {
      uint32_t* words = share_words(args, D);
      for (int b = threadIdx.x; b < a.batch; b += kThreads) words[4 + b] = first[b];
      if (threadIdx.x == 0) words[0] = shares.free, words[1] = shares.large, words[2] = shares.small;
    }
    // neighbouring shares go to different SMs
    const uint32_t number = has_units ? shares.free + warp * busy + blockIdx.x : warp * idle + (blockIdx.x - busy);
    if (shares.size(number) > 0)
      own_worker<D>(&tmap_k16, &tmap_v16, args, bars, first, place, shares, number, base + warp * ring_of<D>() * 16 * D * 4, warp, lane, G);
  }
  __syncthreads();
  if (bars.abort_flag != 0) {
    if (threadIdx.x == 0 && a.status != nullptr && atomicCAS(a.status, 0u, 13u) == 0u) {
      a.status[1] = bars.abort_flag;
      a.status[2] = blockIdx.x;
      a.status[3] = static_cast<uint32_t>(n_units);
    }
    __nanosleep(1000000);   // copies still in flight get a bounded chance to land before the CTA retires
  }
}

// Merges the partial results of a row's heads (a CTA per row and KV head): the weight of every partial result once per head, a warp
// per head, then the sums 16 bytes a lane.
constexpr int kMergeThreads = 128;
template <int D>
__global__ void __launch_bounds__(kMergeThreads)
shared_merge_kernel(XpDecodeSharedArgs args, int G) {
  pdl::wait();
  pdl::release_short();
  constexpr int kMost = XP_PREFIX_PARTS + XP_PREFIX_OWN;
  __shared__ float wt[16][kMost + 1];               // weights, then 1 / sum of weights
  const XpDecodeAttnArgs& a = args.a;
  const int hk = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t* words = share_words(args, D);
  // Everything that does not hang on another load is requested at once: the shares, the pairs of all slots (those that were not
  // written are dropped), and below the sums of the pieces.
  const uint32_t words_free = words[0], words_large = words[1], words_small = words[2], row_first = words[4 + b];
  const int shared = shared_tokens(args, b), most_parts = b < args.plan_rows ? args.row_parts[b] : 0;
  const int parts = shared > 0 ? most_parts : 0, tiles = (row_tokens(args, b) - shared + 15) >> 4;
  const int slots = args.max_parts + args.own_slots;
  float2 pair[4][3];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int g = warp + k * (kMergeThreads / 32);
    const Partials p(args, D, b, hk * G + min(g, G - 1));
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int i = j * 32 + lane;
      pair[k][j] = g < G && i < slots ? p.pairs[i] : make_float2(-CUDART_INF_F, 0.f);
    }
  }
  const Shares cut{words_free, words_large, words_small};
  const uint32_t units = row_units(a), row0 = row_first * units;
  // shares that hold tiles of a unit of this row
  auto shares = [&](int unit) {
    if (tiles == 0) return 0;
    const uint32_t start = row0 + static_cast<uint32_t>(unit) * tiles;
    return static_cast<int>(cut.worker(start + tiles - 1) - cut.worker(start)) + 1;
  };
  const int own0 = shares(units == a.kv_heads ? hk : 2 * hk), own1 = units == a.kv_heads ? 0 : shares(2 * hk + 1);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int g = warp + k * (kMergeThreads / 32), own = g < 8 ? own0 : own1;
    if (g >= G) break;
    float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int i = j * 32 + lane;
      const bool used = i < args.max_parts ? i < parts : i < args.max_parts + own;
      if (!used) pair[k][j] = make_float2(-CUDART_INF_F, 0.f);
      top = fmaxf(top, pair[k][j].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int i = j * 32 + lane;
      const float c = pair[k][j].x == -CUDART_INF_F ? 0.f : exp2f(pair[k][j].x - top);
      if (i < slots) wt[g][i] = c;
      sum = fmaf(pair[k][j].y, c, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) wt[g][kMost] = sum == 0.f ? 0.f : 1.f / sum;      // a row without tokens gives zeros
  }
  __syncthreads();
  for (int i = threadIdx.x * 4; i < G * D; i += kMergeThreads * 4) {
    const int g = i / D, d = i % D, hq = hk * G + g, n = parts + (g < 8 ? own0 : own1);
    const Partials p(args, D, b, hq);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const int at = s < parts ? s : args.max_parts + s - parts;
      const float4 o = *reinterpret_cast<const float4*>(p.sums + static_cast<size_t>(at) * D + d);
      const float c = wt[g][at];
      v[0] = fmaf(o.x, c, v[0]), v[1] = fmaf(o.y, c, v[1]), v[2] = fmaf(o.z, c, v[2]), v[3] = fmaf(o.w, c, v[3]);
    }
    const float c = wt[g][kMost];
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (static_cast<size_t>(b) * a.q_heads + hq) * D + d) =
        make_uint2(pack2(v[0] * c, v[1] * c), pack2(v[2] * c, v[3] * c));
  }
}

// Shared memory above the default is asked for once per device and kernel.
template <typename K>
static int allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -21;
  const uint64_t bit = 1ull << (dev & 63);
  if ((done & bit) == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -21;
    done |= bit;
  }
  return 0;
}

template <int D>
static int launch(const XpDecodeSharedArgs& args, cudaStream_t s) {
  const XpDecodeAttnArgs& a = args.a;
  const int G = a.q_heads / a.kv_heads;
  const uint64_t tokens = static_cast<uint64_t>(a.num_pages) * a.page_size;
  const int box_tokens = a.page_size >= 64 ? 64 : 16;     // a copy brings so many tokens and 64 dims
  CUtensorMap mq, mk, mv, mk16, mv16;
  if (tmap::cache().get_kv(&mk16, a.k_cache, tokens, a.kv_heads, D) != 0 || tmap::cache().get_kv(&mv16, a.v_cache, tokens, a.kv_heads, D) != 0) return -20;
  if (tmap::cache().get_kv(&mk, a.k_cache, tokens, a.kv_heads, D, box_tokens) != 0 || tmap::cache().get_kv(&mv, a.v_cache, tokens, a.kv_heads, D, box_tokens) != 0) return -20;
  if (tmap::cache().get_q(&mq, a.q, static_cast<uint64_t>(a.batch), a.q_heads, D, G, kRows / G) != 0) return -20;
  constexpr int kTiles = 2 * (D / 64) * kRows * 128 + kStages * 2 * (D / 64) * kBN * 128, kRings = kWarps * ring_of<D>() * 16 * D * 4;
  constexpr int kSmem = (kTiles > kRings ? kTiles : kRings) + (2 * XP_PREFIX_ROWS + 1) * 4 + 1024;
  static_assert(kSmem + sizeof(Bars) <= 227 * 1024, "tiles exceed the shared memory of an SM");
  static std::atomic<uint64_t> allowed{0};
  if (const int rc = allow_smem(shared_prefix_kernel<D>, kSmem, allowed); rc != 0) return rc;
  pdl::launch(shared_prefix_kernel<D>, 148, kThreads, kSmem, s, 1, mq, mk, mv, mk16, mv16, args, G, box_tokens);
  pdl::launch(shared_merge_kernel<D>, dim3(a.kv_heads, a.batch), kMergeThreads, 0, s, 1, args, G);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}

}  // namespace prefix
}  // namespace xpool

extern "C" int xp_decode_shared(const XpDecodeSharedArgs* r, void* stream) {
  const XpDecodeAttnArgs* a = &r->a;
  if (a->batch <= 0) return 0;
  if (r->max_pieces <= 0) {                                      // no prefixes
    XpDecodeAttnArgs plain = *a;
    plain.max_len = r->max_len > 0 ? r->max_len : -1;
    return xp_decode_attn(&plain, stream);
  }
  if (a->kv_heads <= 0 || a->q_heads % a->kv_heads != 0) return -10;
  if (a->ws == nullptr || (reinterpret_cast<uintptr_t>(a->ws) & 15) != 0 || (reinterpret_cast<uintptr_t>(a->out) & 7) != 0) return -11;
  if (a->q_heads / a->kv_heads > 16 || a->num_pages <= 0 || a->page_size < 16 || (a->page_size & (a->page_size - 1)) != 0 ||
      (reinterpret_cast<uintptr_t>(a->q) & 15) != 0)
    return -12;
  if (a->batch > XP_PREFIX_ROWS || r->max_parts < 1 || r->max_parts > XP_PREFIX_PARTS || r->own_slots < 2 || r->own_slots > XP_PREFIX_OWN) return -13;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->head_dim == 128) return xpool::prefix::launch<128>(*r, s);
  if (a->head_dim == 64) return xpool::prefix::launch<64>(*r, s);
  return -14;
}
