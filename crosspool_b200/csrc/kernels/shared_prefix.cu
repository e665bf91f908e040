// Attention of query rows over a prefix that they share, on the Blackwell tensor cores. A plan cuts every prefix into pieces (a
// range of its tokens, and up to 2 x (128 / G) consecutive rows that read it, G query heads to a KV head); a piece leaves partial
// results, un-normalised sums O = sum_t 2^(s_t - m) v_t with their maximum m and sum of weights l, to which the decode kernel
// (attn_decode.cu) adds the tokens of each row's own. With M rows of queries on a prefix the keys and values of a KV head are
// multiplied by M G queries once they are in shared memory, where row by row attention reads them M times.
//
// A persistent CTA per SM takes (piece, KV head) units in turn: two tiles of 128 queries (row of a tile = row * G + head), both
// multiplied against the same 64-token K/V tiles, so that the tensor pipe works on one while the softmax of the other runs.
//
//   warps 0-3   softmax of tile A: thread = query = TMEM lane. Reads its row of S with tcgen05.ld, keeps a running maximum and
//               sum, writes P (bf16) over the start of S as the A operand of the second product, rescales O in tensor memory only
//               when the maximum grew by more than 2^8 (sum and result carry the same stale maximum), and stores the partial result.
//   warps 4-7   the same for tile B.
//   warp 8      TMA producer: Q tiles once a unit, then a ring of K/V tiles through the leader's page table (128-byte swizzle).
//   warp 9      allocates tensor memory and issues every tcgen05.mma: S_A(t+1), PV_A(t), S_B(t+1), PV_B(t).
//
// P is rounded to bf16 for the second product (2^-8 of a weight at most, as in prefill attention); l sums the unrounded weights.
// The last tile of a prefix may end inside its 64 tokens: scores behind the end are selected away and the values zeroed, whatever
// the cache holds there. No other masks: a row that does not see the whole prefix is none of the decode kernel's sharing rows.
// Every wait is bounded; one that runs out sets the abort word, the status word (13) and ends the CTA behind a common barrier.
#include <math_constants.h>

#include "xpool/pdl.cuh"
#include "xpool/request_api.h"
#include "xpool/sm100.cuh"
#include "xpool/tensormap.hpp"

namespace xpool {
namespace prefix {

constexpr int kRows = 128;       // queries of a tile (UMMA M)
constexpr int kBN = 64;          // tokens of a K/V tile
constexpr int kStages = 3;
constexpr int kThreads = 320;
constexpr float kRescaleStep = 8.0f;   // log2 units

struct __align__(8) Bars {
  uint64_t q_full, q_empty;
  uint64_t kv_full[kStages];
  uint64_t kv_empty[kStages];
  uint64_t s_full[2][2];
  uint64_t p_full[2];
  uint64_t pv_done[2];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

// Bounded wait of a converged warp that also gives up when another role of the CTA has; one answer for all lanes.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* b, uint32_t site) {
  bool ok = sm100::mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t deadline = sm100::global_timer_ns() + sm100::kPipelineWaitNs;
    uint32_t spins = 0;
    while (!(ok = sm100::mbar_try_wait(bar, parity))) {
      if ((++spins & 0xffu) == 0) {
        if (b->abort_flag != 0) break;
        if (sm100::global_timer_ns() > deadline) {
          b->abort_flag = site;
          break;
        }
      }
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

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                     const __grid_constant__ XpDecodeSharedArgs args, int G, int box_tokens) {
  constexpr int kHalves = D / 64;                 // 64-dim (128-byte) column blocks of a row
  constexpr int kQHalf = kRows * 128;
  constexpr int kQTile = kHalves * kQHalf;
  constexpr int kKVHalf = kBN * 128;
  constexpr int kKTile = kHalves * kKVHalf;
  constexpr int kStage = 2 * kKTile;              // K then V
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kOCol = 4 * kBN;             // S: two buffers per tile; O_A behind them, then O_B
  extern __shared__ uint8_t smem_dyn[];
  __shared__ Bars bars;

  pdl::wait();
  const XpDecodeAttnArgs& a = args.a;
  const int n_units = min(*args.n_pieces, args.max_pieces) * a.kv_heads;
  const int np = kRows / G;                       // rows of a tile; its last 128 - np G queries are none
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (sm100::smem_u32(smem_dyn) + 1023u) & ~1023u;
  const uint32_t q_s = base, kv_s = base + 2 * kQTile;

  if (threadIdx.x == 0) {
    sm100::mbar_init(&bars.q_full, 1);
    sm100::mbar_init(&bars.q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      sm100::mbar_init(&bars.kv_full[s], 1);
      sm100::mbar_init(&bars.kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      sm100::mbar_init(&bars.s_full[x][0], 1);
      sm100::mbar_init(&bars.s_full[x][1], 1);
      sm100::mbar_init(&bars.p_full[x], 4);
      sm100::mbar_init(&bars.pv_done[x], 1);
    }
    bars.abort_flag = 0;
    sm100::mbar_fence_init();
    sm100::fence_proxy_async_smem();
  }
  if (warp == 9) {
    sm100::tmem_alloc(&bars.tmem_base, kTmemCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before_sync();
  __syncthreads();
  sm100::tc_fence_after_sync();
  const uint32_t tmem = bars.tmem_base;
  pdl::release();

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    const int page_shift = 31 - __clz(a.page_size), page_mask = a.page_size - 1;
    const int boxes = kBN / box_tokens, box_bytes = box_tokens * 128;
    const uint32_t q_bytes = static_cast<uint32_t>(2 * kHalves * np * G * 128);
    int it = 0, ord = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < n_units; u += gridDim.x, ++ord) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int hk = u % a.kv_heads;
      const int* table = a.block_table + static_cast<size_t>(p.leader) * a.max_blocks;
      if (ord > 0 && !wait_bar(&bars.q_empty, (ord - 1) & 1, &bars, 1)) break;
      if (lane == 0) sm100::mbar_arrive_expect_tx(&bars.q_full, q_bytes);
      __syncwarp();
      if (lane < 2 * kHalves) {
        const int x = lane / kHalves, h = lane % kHalves;
        sm100::tma_load_3d_addr(q_s + x * kQTile + h * kQHalf, &tmap_q, sm100::smem_u32(&bars.q_full), h * 64, hk * G, p.row0 + x * np);
      }
      const int n_tiles = (p.tok1 - p.tok0 + kBN - 1) / kBN;
      for (int t = 0; t < n_tiles; ++t, ++it) {
        const int s = it % kStages;
        if (it >= kStages && !(ok = wait_bar(&bars.kv_empty[s], ((it / kStages) - 1) & 1, &bars, 2))) break;
        if (lane == 0) sm100::mbar_arrive_expect_tx(&bars.kv_full[s], kStage);
        __syncwarp();
        const uint32_t full = sm100::smem_u32(&bars.kv_full[s]), dst = kv_s + s * kStage;
        if (boxes == 1) {
          if (lane < 2) {
            const int tk = p.tok0 + t * kBN;
            const int tok = (table[tk >> page_shift] << page_shift) + (tk & page_mask);
            sm100::tma_load_4d_addr(dst + lane * kKTile, lane ? &tmap_v : &tmap_k, full, 0, tok, 0, hk);
          }
        } else if (lane < 2 * boxes * kHalves) {
          const int h = lane % kHalves, is_v = (lane / kHalves) & 1, j = lane / (2 * kHalves);
          // boxes behind the end repeat the last one
          const int tk = min(p.tok0 + t * kBN + j * box_tokens, (p.tok1 - 1) & ~(box_tokens - 1));
          const int tok = (table[tk >> page_shift] << page_shift) + (tk & page_mask);
          sm100::tma_load_3d_addr(dst + is_v * kKTile + h * kKVHalf + j * box_bytes, is_v ? &tmap_v : &tmap_k, full, h * 64, hk, tok);
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer (the whole warp walks, one elected lane issues)
    const bool leader = sm100::elect_one();
    const uint32_t idesc_s = sm100::umma_idesc_bf16(kRows, kBN);
    const uint32_t idesc_o = sm100::umma_idesc_bf16_bmn(kRows, D);
    int it = 0, ord = 0, count[2] = {0, 0};       // K/V tiles; units; tiles that query tile A (B) has multiplied
    auto issue_s = [&](int x, int i, int c) {     // S_x = Q_x K(i)^T into buffer c & 1
      if (!leader) return;
      const uint32_t d = tmem + static_cast<uint32_t>((x * 2 + (c & 1)) * kBN);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint64_t da = sm100::umma_desc_sw128(q_s + x * kQTile + (ks >> 2) * kQHalf) + (ks & 3) * 2;
        const uint64_t db = sm100::umma_desc_sw128(kv_s + (i % kStages) * kStage + (ks >> 2) * kKVHalf) + (ks & 3) * 2;
        sm100::umma_bf16(d, da, db, idesc_s, ks > 0 ? 1u : 0u);
      }
      sm100::umma_commit(&bars.s_full[x][c & 1]);
    };
    auto issue_pv = [&](int x, int i, int c, bool more) {   // O_x (+)= P_x V(i)
      if (!leader) return;
      const uint32_t d = tmem + kOCol + static_cast<uint32_t>(x * D);
#pragma unroll
      for (int kk = 0; kk < kBN / 16; ++kk) {
        const uint64_t db = sm100::umma_desc_mn_sw128(kv_s + (i % kStages) * kStage + kKTile + kk * 2048, kKVHalf, 1024);
        // P sits in the first 32 columns of the S buffer it was computed from, 8 columns per K step
        sm100::umma_bf16_ts(d, tmem + static_cast<uint32_t>((x * 2 + (c & 1)) * kBN + kk * 8), db, idesc_o, (more || kk > 0) ? 1u : 0u);
      }
      sm100::umma_commit(&bars.pv_done[x]);
    };
    bool ok = true;
    for (int u = blockIdx.x; ok && u < n_units; u += gridDim.x, ++ord) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int n_tiles = (p.tok1 - p.tok0 + kBN - 1) / kBN, tiles_x = p.rows > np ? 2 : 1;
      ok = wait_bar(&bars.q_full, ord & 1, &bars, 3) && wait_bar(&bars.kv_full[it % kStages], (it / kStages) & 1, &bars, 4);
      if (!ok) break;
      sm100::tc_fence_after_sync();
      for (int x = 0; x < tiles_x; ++x) issue_s(x, it, count[x]);
      if (n_tiles == 1 && leader) sm100::umma_commit(&bars.q_empty);
      for (int t = 0; ok && t < n_tiles; ++t) {
        const bool next = t + 1 < n_tiles;
        const int i = it + t;
        if (next) ok = wait_bar(&bars.kv_full[(i + 1) % kStages], ((i + 1) / kStages) & 1, &bars, 5);
        for (int x = 0; ok && x < tiles_x; ++x) {
          const int c = count[x];
          if (next) {
            sm100::tc_fence_after_sync();
            issue_s(x, i + 1, c + 1);
            if (t + 2 == n_tiles && x + 1 == tiles_x && leader) sm100::umma_commit(&bars.q_empty);   // the unit's last use of Q
          }
          ok = wait_bar(&bars.p_full[x], c & 1, &bars, 6);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          issue_pv(x, i, c, t > 0);
          count[x] = c + 1;
        }
        if (ok && leader) sm100::umma_commit(&bars.kv_empty[i % kStages]);
      }
      it += n_tiles;
    }
  } else {
    // ------------------------------------------------------------------ softmax and partial results (warps 0-7)
    const int x = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int pos = row / G, head = row % G;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_t = tmem + lane_off + kOCol + static_cast<uint32_t>(x * D);
    const float sc2 = a.scale * 1.4426950408889634f;
    const int slots = args.max_parts + (a.num_splits > 1 ? a.num_splits : 0);
    int it = 0, c = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < n_units; u += gridDim.x) {
      const XpPrefixPiece p = args.pieces[u / a.kv_heads];
      const int n_tiles = (p.tok1 - p.tok0 + kBN - 1) / kBN;
      if (x == 0 || p.rows > np) {
        float m_used = -CUDART_INF_F, l = 0.f;
        for (int t = 0; t < n_tiles; ++t, ++c) {
          ok = wait_bar(&bars.s_full[x][c & 1], (c >> 1) & 1, &bars, 7);
          if (!ok) break;
          sm100::tc_fence_after_sync();
          uint32_t sv[kBN];
          const uint32_t s_t = tmem + lane_off + static_cast<uint32_t>((x * 2 + (c & 1)) * kBN);
          sm100::tmem_ld32_issue(s_t, sv);
          sm100::tmem_ld32_issue(s_t + 32, sv + 32);
          sm100::tmem_ld_wait_all(sv);
          sm100::tmem_ld_wait_all(sv + 32);
          const int nvis = p.tok1 - p.tok0 - t * kBN;       // tokens of the prefix in this tile (a uniform number)
          if (nvis < kBN) {
#pragma unroll
            for (int j = 0; j < kBN; ++j)
              if (j >= nvis) sv[j] = 0xff800000u;           // -inf: selected, never computed with
          }
          float mx4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int j = 0; j < kBN; j += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx4[e] = max3(mx4[e], __uint_as_float(sv[j + 2 * e]), __uint_as_float(sv[j + 2 * e + 1]));
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
          float sum4[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t pk[kBN / 2];
#pragma unroll
          for (int j = 0; j < kBN; j += 2) {
            const float p0 = sm100::ex2_approx(fmaf(__uint_as_float(sv[j]), sc2, -m_sub));
            const float p1 = sm100::ex2_approx(fmaf(__uint_as_float(sv[j + 1]), sc2, -m_sub));
            sum4[(j >> 1) & 3] += p0 + p1;
            pk[j >> 1] = pack2(p0, p1);
          }
          l = l * factor + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
          const bool rescale = t > 0 && __any_sync(0xffffffffu, factor != 1.f);
          if (rescale) {
            // the previous second product must have retired: it accumulates into O
            ok = wait_bar(&bars.pv_done[x], (c - 1) & 1, &bars, 8);
            if (!ok) break;
            sm100::tc_fence_after_sync();
#pragma unroll 1
            for (int e = 0; e < D; e += 32) {
              uint32_t ov[32];
              sm100::tmem_ld32_issue(o_t + e, ov);
              sm100::tmem_ld_wait_all(ov);
#pragma unroll
              for (int j = 0; j < 32; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * factor);
              sm100::tmem_st32(o_t + e, ov);
            }
            sm100::tmem_st_wait();
          }
          // P as the tensor core's A operand: 32 columns of two bf16 each, over the start of the S buffer
          sm100::tmem_st32(s_t, pk);
          if (nvis < kBN && x == 0) {
            // cache slots behind the prefix may hold anything: zero those V rows (a weight of zero times NaN). Tile A's product
            // is issued before tile B's, and both read this stage.
            const uint32_t v_s = kv_s + ((it + t) % kStages) * kStage + kKTile;
            for (int i = row; i < (kBN - nvis) * (D / 8); i += kRows) {
              const int R = nvis + i / (D / 8), cc = i % (D / 8);
              const uint32_t off = (cc >> 3) * kKVHalf + R * 128 + (((cc & 7) ^ (R & 7)) << 4);
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_s + off), "r"(0u) : "memory");
            }
            sm100::fence_proxy_async_smem();
          }
          sm100::tmem_st_wait();
          sm100::tc_fence_before_sync();
          // every phase of pv_done is consumed in order, before the arrival below lets the next one complete
          if (t > 0 && !rescale) {
            ok = wait_bar(&bars.pv_done[x], (c - 1) & 1, &bars, 9);
            if (!ok) break;
          }
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&bars.p_full[x]);
        }
        if (ok) ok = wait_bar(&bars.pv_done[x], (c - 1) & 1, &bars, 10);
        if (ok) {
          sm100::tc_fence_after_sync();
          const int r = x * np + pos;
          const bool stored = pos < np && r < p.rows;
          const int hq = (u % a.kv_heads) * G + head;
          const size_t at = (static_cast<size_t>(p.row0 + (stored ? r : 0)) * a.q_heads + hq) * slots + p.part;
#pragma unroll 1
          for (int e = 0; e < D; e += 32) {
            uint32_t ov[32];
            sm100::tmem_ld32_issue(o_t + e, ov);
            sm100::tmem_ld_wait_all(ov);
            if (stored) {
              uint4* o = reinterpret_cast<uint4*>(a.ws + at * D + e);
#pragma unroll
              for (int j = 0; j < 32; j += 4) o[j / 4] = make_uint4(ov[j], ov[j + 1], ov[j + 2], ov[j + 3]);
            }
          }
          if (stored)
            *reinterpret_cast<float2*>(a.ws + static_cast<size_t>(a.batch) * a.q_heads * slots * D + at * 2) = make_float2(m_used, l);
          sm100::tc_fence_before_sync();       // O has been read before the next unit's first arrival at p_full
        }
      }
      it += n_tiles;
    }
  }
  // ------------------------------------------------------------------ common exit
  sm100::tc_fence_before_sync();
  __syncthreads();
  if (bars.abort_flag != 0) {
    if (threadIdx.x == 0 && a.status != nullptr && atomicCAS(a.status, 0u, 13u) == 0u) {
      a.status[1] = bars.abort_flag;
      a.status[2] = blockIdx.x;
      a.status[3] = static_cast<uint32_t>(n_units);
    }
    __nanosleep(1000000);   // copies still in flight get a bounded chance to land before the CTA retires
  }
  if (warp == 9) {
    sm100::tc_fence_after_sync();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
}

// Shared memory above the default is asked for once per device and kernel.
template <typename K>
static int allow_smem(K kernel, int bytes, uint64_t& done) {
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
  const int box_tokens = a.page_size >= kBN ? kBN : 16;   // one copy brings a whole K (or V) tile, or 16 tokens and 64 dims
  CUtensorMap mq, mk, mv;
  if (box_tokens == kBN) {
    if (tmap::cache().get_kv4(&mk, a.k_cache, tokens, a.kv_heads, D, kBN) != 0 || tmap::cache().get_kv4(&mv, a.v_cache, tokens, a.kv_heads, D, kBN) != 0) return -20;
  } else {
    if (tmap::cache().get_kv(&mk, a.k_cache, tokens, a.kv_heads, D) != 0 || tmap::cache().get_kv(&mv, a.v_cache, tokens, a.kv_heads, D) != 0) return -20;
  }
  if (tmap::cache().get_q(&mq, a.q, static_cast<uint64_t>(a.batch), a.q_heads, D, G, kRows / G) != 0) return -20;
  constexpr int kSmem = 2 * (D / 64) * kRows * 128 + kStages * 2 * (D / 64) * kBN * 128 + 1024;
  static uint64_t allowed = 0;
  if (const int rc = allow_smem(shared_prefix_kernel<D>, kSmem, allowed); rc != 0) return rc;
  const int units = args.max_pieces * a.kv_heads;
  pdl::launch(shared_prefix_kernel<D>, units < 148 ? units : 148, kThreads, kSmem, s, 1, mq, mk, mv, args, G, box_tokens);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}

}  // namespace prefix
}  // namespace xpool

// Launches the pieces of a plan (xp_decode_shared has checked the arguments).
extern "C" int xp_shared_prefix_pieces(const XpDecodeSharedArgs* r, void* stream) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return r->a.head_dim == 128 ? xpool::prefix::launch<128>(*r, s) : xpool::prefix::launch<64>(*r, s);
}
