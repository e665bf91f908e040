// Low-rank adapters of many requests beside a shared projection: out[r] = y[r] + scale (B (A x[r])), every row with the A, B and
// scale of its own adapter. A plan's items are up to 16 rows of one adapter; a cluster of CTAs takes an item:
//
//   h = x A^T      the CTAs share k, the warps of a CTA its blocks of 32; partial sums meet in shared memory, then in the
//                  distributed shared memory of the cluster, always in the same order
//   out = y + scale h B^T    the CTAs share the features, their warps blocks of 32
//
// Both products by mma.m16n8k16 with the rows as M. An adapter is read once for 16 rows or fewer: 32 flop a byte at most, far
// below what the tensor pipe needs, so what counts is bytes in flight and the one exchange between the products. Every lane copies
// its own fragments to shared memory and needs no barrier for them: the order of a sum's terms is free, so a lane's operand of two
// steps of k are 8 neighbouring elements (16 bytes) of a row of x or A, and the columns of four tiles of features are dealt so that
// a lane holds 8 neighbouring features of y and out. A and B lie in the order of the lanes, so that a copy of a warp is 512 bytes in
// a row (eight rows of 64 bytes, or 32, before: 2000 rows of ranks 120 and 128 beside 4096 -> 4096 took 67 us, then 47). While the first
// product runs, B and y are brought to the L2.
//
// h enters the second product as a bf16 pair (high and low part, 16 mantissa bits): its rounding to bf16 alone would be as large as
// the result's. Sums are fp32.
#include <cooperative_groups.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "xpool/mma_sync.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace lora {

using bf16 = __nv_bfloat16;
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxRank = 128;
constexpr int kItemRows = 16;
constexpr int kMaxCluster = 8;
constexpr int kPitch = 64 + 4;                       // fp32 row of a warp's partial sums

// 16 bytes to shared memory; zeros when not ok
__device__ __forceinline__ void copy16(uint32_t dst, const bf16* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// (kept in the L1: other warps of the CTA read the same)
__device__ __forceinline__ void copy16_kept(uint32_t dst, const bf16* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most `left` of the groups issued last are in flight
__device__ __forceinline__ void landed(int left) {
  if (left >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {      // whole 16 bytes
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
// 16 bytes to the shared memory of a CTA of the cluster
__device__ __forceinline__ void st_cluster(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, const uint4& v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void add4(float4& s, const float4& v) { s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w; }

// A warp's ring, and its partial sums between the products. 10 KB: four blocks of k of three tiles, and two CTAs to an SM.
template <int kTiles>
constexpr int region_bytes() { return kTiles == 4 ? 10240 : 15360; }
static_assert(kItemRows * kPitch * 4 <= region_bytes<4>() && (2 + 8) * 512 * 3 <= region_bytes<8>() && 1024 + kMaxRank * 64 <= region_bytes<4>(), "region");

// Shared memory: the warps' regions; the sums of all CTAs for the blocks of 16 ranks that this CTA adds up, [blocks][CTA]
// [16 rows][16 ranks]; the whole h as fragments, 8 words per lane and block.
__host__ __device__ constexpr int smem_bytes(int all_ranks, int ranks, int region) {
  return kWarps * region + (all_ranks / 16 + ranks - 1) / ranks * ranks * 1024 + all_ranks / 16 * 1024;
}

// kTiles: tiles of 8 ranks that a warp of the first product takes, at most; four are enough for 256 columns of h.
template <int kTiles>
__global__ void __launch_bounds__(kThreads, 2)
lora_kernel(XpLoraArgs a, int ranks) {
  namespace cg = cooperative_groups;
  // another CTA's shared memory is written once that CTA is known to have started
  auto started = cg::this_cluster().barrier_arrive();
  pdl::wait();
  pdl::release();
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kRegion = region_bytes<kTiles>();
  float* sums = reinterpret_cast<float*>(smem + kWarps * kRegion);
  uint4* frags = reinterpret_cast<uint4*>(sums + (a.parts * a.rank / 16 + ranks - 1) / ranks * ranks * 256);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint32_t ring = sm100::smem_u32(smem) + warp * kRegion + lane * 16;
  const int rank = blockIdx.x % ranks, first_item = blockIdx.x / ranks, step = gridDim.x / ranks;
  XpLoraItem item = a.items[first_item];            // (the grid has no more clusters than items)
  const int n_items = min(*a.n_items, a.max_items);
  bool met = false;                                  // the CTAs of the cluster have all started

  for (int it = first_item; it < n_items; it += step) {
    if (it != first_item) item = a.items[it];
    const int slot = item.slot, rk = slot >= 0 && slot < a.slots ? a.ranks[slot] : 0;
    // rows of this lane: g and g + 8 of the item
    const bool on0 = g < item.rows, on1 = g + 8 < item.rows;
    const int r0 = on0 ? a.perm[item.first + g] : 0, r1 = on1 ? a.perm[item.first + g + 8] : 0;
    const bf16* y = reinterpret_cast<const bf16*>(a.y);
    bf16* out = reinterpret_cast<bf16*>(a.out);
    // features of this CTA, in blocks of 32 that do not cross parts
    int blocks = 0;
#pragma unroll
    for (int p = 0; p < XP_LORA_PARTS; ++p)
      if (p < a.parts) blocks += (a.part_end[p] - (p ? a.part_end[p - 1] : 0) + 31) >> 5;
    const int b0 = static_cast<int>(static_cast<long long>(blocks) * rank / ranks), b1 = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / ranks);
    auto locate = [&](int b, int& p, int& f, int& end) {      // part of a block, its first feature, the part's end
      int begin = 0;
      p = 0;
      while (true) {
        const int n = (a.part_end[p] - begin + 31) >> 5;
        if (b < n || p + 1 == a.parts) break;
        b -= n, begin = a.part_end[p], ++p;
      }
      f = begin + b * 32, end = a.part_end[p];
    };
    if (rk == 0) {                                   // no adapter: the rows are copied
      if (a.out != a.y) {
        for (int b = b0 + warp; b < b1; b += kWarps) {
          int p, f, end;
          locate(b, p, f, end);
          f += q * 8;
          if (f >= end) continue;
          if (on0) *reinterpret_cast<uint4*>(out + static_cast<size_t>(r0) * a.ld_out + f) = *reinterpret_cast<const uint4*>(y + static_cast<size_t>(r0) * a.ld_y + f);
          if (on1) *reinterpret_cast<uint4*>(out + static_cast<size_t>(r1) * a.ld_out + f) = *reinterpret_cast<const uint4*>(y + static_cast<size_t>(r1) * a.ld_y + f);
        }
      }
      continue;                                      // (the same for all CTAs of the cluster)
    }
    const bf16* bw = reinterpret_cast<const bf16*>(a.b) + static_cast<size_t>(slot) * a.n * a.rank;
    // ---- h = x A^T, this CTA's share of k
    const int kblocks = (a.k + 31) >> 5;
    const int k0 = static_cast<int>(static_cast<long long>(kblocks) * rank / ranks), k1 = static_cast<int>(static_cast<long long>(kblocks) * (rank + 1) / ranks);
    const bf16* x = reinterpret_cast<const bf16*>(a.x);
    const bf16* aw = reinterpret_cast<const bf16*>(a.a) + static_cast<size_t>(slot) * a.parts * a.rank * kblocks * 32;
    auto prefetch_second = [&]() {                   // B and y of the second product, to the L2
      int p, f, end, f1;
      locate(b1 - 1, p, f1, end);
      f1 = min(f1 + 32, end);
      locate(b0, p, f, end);
      const uint32_t bytes = static_cast<uint32_t>(f1 - f) * rk * 2;
      for (uint32_t at = lane * 4096u; at < bytes; at += 32 * 4096u)
        prefetch_l2(reinterpret_cast<const uint8_t*>(bw + static_cast<size_t>(f) * rk) + at, min(4096u, bytes - at));
      if (lane < item.rows) prefetch_l2(y + static_cast<size_t>(a.perm[item.first + lane]) * a.ld_y + f, static_cast<uint32_t>(f1 - f) * 2);
    };
    // The warps share the columns of h in groups of kTiles tiles, and those of a group its blocks of k.
    const int all = a.parts * rk, n_tiles = all >> 3;   // columns of h, part after part
    const int groups = n_tiles <= kTiles ? 1 : n_tiles <= 2 * kTiles ? 2 : n_tiles <= 4 * kTiles ? 4 : 8, each = kWarps / groups;
    const int per = (n_tiles + groups - 1) / groups, t0 = warp / each * per, tiles = max(0, min(per, n_tiles - t0));
    // (the steps are bound by their instructions: NT > 0 is a known number of tiles, which may lie side by side in one part)
    auto first_product = [&](auto known, auto side_by_side) {
      constexpr int NT = decltype(known)::value, kMost = NT > 0 ? NT : kTiles;
      constexpr bool kBeside = decltype(side_by_side)::value;
      float acc[kMost][4];
      const bf16* wrow[kBeside ? 1 : kMost];
#pragma unroll
      for (int t = 0; t < kMost; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
      for (int t = 0; t < (kBeside ? 1 : kMost); ++t) {
        const int c = (t0 + min(t, tiles - 1)) * 8;
        wrow[t] = aw + static_cast<size_t>(c / rk) * a.rank * kblocks * 32 + (c % rk >> 3) * 256 + lane * 8;
      }
      const uint32_t stage = (2 + (NT > 0 ? NT : tiles)) * 512;
      const int depth = min(4, static_cast<int>(kRegion / stage));
      const bf16* x0 = x + static_cast<size_t>(r0) * a.ldx + q * 8;
      const bf16* x1 = x + static_cast<size_t>(r1) * a.ldx + q * 8;
      const int k_left = a.k - q * 8;                // blocks that begin before it have elements of this lane
      auto issue = [&](int kb, uint32_t to) {
        if (kb < k1) {
          const bool in = kb * 32 < k_left;
          const int at = in ? kb * 32 : 0;
          const size_t w_at = static_cast<size_t>(kb) * (a.rank * 32);
          copy16_kept(to, x0 + (in ? at : -q * 8), in && on0);
          copy16_kept(to + 512, x1 + (in ? at : -q * 8), in && on1);
          if constexpr (kBeside) {
            const bf16* from = wrow[0] + w_at;
#pragma unroll
            for (int t = 0; t < NT; ++t) copy16(to + 1024 + t * 512, from + t * 256, true);
          } else {
#pragma unroll
            for (int t = 0; t < kMost; ++t)
              if (NT > 0 || t < tiles) copy16(to + 1024 + t * 512, wrow[t] + w_at, true);
          }
        }
        issued();
      };
      const int kb0 = k0 + warp % each;
      for (int i = 0; i < depth; ++i) issue(kb0 + i * each, ring + i * stage);
      if (warp == 0 && b1 > b0) prefetch_second();
      uint32_t at = ring;
      for (int kb = kb0; kb < k1; kb += each) {
        landed(depth - 1);
        const uint4 u = lds16(at), v = lds16(at + 512);
        const uint32_t lo[4] = {u.x, v.x, u.y, v.y}, hi[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
        for (int t = 0; t < kMost; ++t)
          if (NT > 0 || t < tiles) {
            const uint4 w = lds16(at + 1024 + t * 512);
            frag::mma(acc[t], lo, w.x, w.y);
            frag::mma(acc[t], hi, w.z, w.w);
          }
        issue(kb + depth * each, at);
        at = at + stage == ring + depth * stage ? ring : at + stage;
      }
      landed(0);
      __syncwarp();                                  // the partial sums lie over all lanes' copies
      float* mine = reinterpret_cast<float*>(smem + warp * kRegion) + g * kPitch + q * 2;
#pragma unroll
      for (int t = 0; t < kMost; ++t)
        if (NT > 0 || t < tiles) {
          *reinterpret_cast<float2*>(mine + t * 8) = make_float2(acc[t][0], acc[t][1]);
          *reinterpret_cast<float2*>(mine + 8 * kPitch + t * 8) = make_float2(acc[t][2], acc[t][3]);
        }
    };
    if (tiles > 0) {
      const bool beside = t0 * 8 / rk == (t0 + tiles - 1) * 8 / rk;
      if (tiles == (kTiles == 4 ? 3 : 6)) first_product(std::integral_constant<int, kTiles == 4 ? 3 : 6>(), std::false_type());
      else if (beside && tiles == 4) first_product(std::integral_constant<int, 4>(), std::true_type());
      else if (beside && tiles == 2) first_product(std::integral_constant<int, 2>(), std::true_type());
      else first_product(std::integral_constant<int, 0>(), std::false_type());
    }
    __syncthreads();
    if (!met) {
      cg::this_cluster().barrier_wait(std::move(started));
      met = true;
    }
    // ---- the cluster's sums: every block of 16 ranks has a CTA that adds up what all have of it and hands the fragments round
    const uint32_t sums_addr = sm100::smem_u32(sums), frags_addr = sm100::smem_u32(frags);
    for (int i = threadIdx.x; i < kItemRows * all / 4; i += kThreads) {
      const int r = i / (all / 4), c = i % (all / 4) * 4, gr = (c >> 3) / per, kb = c >> 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = gr * each; w < (gr + 1) * each; ++w) add4(s, *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * kRegion) + r * kPitch + c - gr * per * 8));
      st_cluster(sm100::map_rank(sums_addr, kb % ranks) + static_cast<uint32_t>((kb / ranks * ranks + rank) * 1024 + r * 64 + (c & 15) * 4), s);
    }
    sm100::cluster_sync();
    // ---- the first blocks of the second product are on their way
    const uint32_t stage = 1024 + rk * 64;             // y, and 16 bytes per two tiles and block of ranks
    const int depth = min(4, static_cast<int>(kRegion / stage));
    auto issue = [&](int b, int s) {
      if (b < b1) {
        int p, f, end;
        locate(b, p, f, end);
        const int fl = f + q * 8;                      // this lane's features of y and out
        const bool in = fl < end;
        copy16(ring + s * stage, y + static_cast<size_t>(r0) * a.ld_y + (in ? fl : f), in && on0);
        copy16(ring + s * stage + 512, y + static_cast<size_t>(r1) * a.ld_y + (in ? fl : f), in && on1);
        // column g of tile t is feature (g / 2) * 8 + 2 t + g % 2 of the block
        const int eights = min(4, (end - f) >> 3);
        const bool ing = g >> 1 < eights;
        const bf16* brow = bw + static_cast<size_t>(f) * rk + (ing ? lane * 8 : 0);
        if (eights == 4) {
#pragma unroll 4
          for (int i = 0; i < rk >> 3; ++i) copy16(ring + s * stage + 1024 + i * 512, brow + i * 256, true);
        } else {
          for (int i = 0; i < rk >> 3; ++i) copy16(ring + s * stage + 1024 + i * 512, brow + i * eights * 64, ing);
        }
      }
      issued();
    };
    for (int i = 0; i < depth; ++i) issue(b0 + warp + i * kWarps, i);
    for (int i = threadIdx.x; i < (all / 16 - rank + ranks - 1) / ranks * 32; i += kThreads) {
      // lane (g, q) of a block holds ranks 4 q .. 4 q + 3 of rows g and g + 8
      const int kb = i >> 5, l = i & 31;
      const float* from = sums + kb * ranks * 256 + (l >> 2) * 16 + (l & 3) * 4;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
      for (int s = 0; s < ranks; ++s) {
        add4(u, *reinterpret_cast<const float4*>(from + s * 256));
        add4(v, *reinterpret_cast<const float4*>(from + s * 256 + 128));
      }
      // Ranks behind a part's own are zero, whatever zeros times x gave; an infinity has no low part.
      const int col = (kb * ranks + rank) * 16, over = a.part_ranks[slot * XP_LORA_PARTS + col / rk] - col % rk - (l & 3) * 4;
      if (over < 4) {
        if (over < 1) u.x = v.x = 0.f;
        if (over < 2) u.y = v.y = 0.f;
        if (over < 3) u.z = v.z = 0.f;
        u.w = v.w = 0.f;
      }
      uint4 hi, lo;
      auto split2 = [](float e, float f, uint32_t& h, uint32_t& low) {
        frag::split2(e, f, h, low);
        if (isinf(e)) low &= 0xffff0000u;
        if (isinf(f)) low &= 0x0000ffffu;
      };
      split2(u.x, u.y, hi.x, lo.x);
      split2(v.x, v.y, hi.y, lo.y);
      split2(u.z, u.w, hi.z, lo.z);
      split2(v.z, v.w, hi.w, lo.w);
      const uint32_t to = frags_addr + static_cast<uint32_t>((kb * ranks + rank) * 32 + l) * 32u;
      for (int s = 0; s < ranks; ++s) {
        const uint32_t at = sm100::map_rank(to, s);
        st_cluster(at, hi);
        st_cluster(at + 16, lo);
      }
    }
    sm100::cluster_sync();                           // nobody reads or writes another CTA's memory behind this

    // ---- out = y + scale h B^T
    const float scale = a.scale[slot];
    int s = 0;
    for (int b = b0 + warp; b < b1; b += kWarps) {
      int p, f, end;
      locate(b, p, f, end);
      const int fl = f + q * 8;
      const bool in = fl < end;
      landed(depth - 1);
      const uint32_t at = ring + s * stage;
      const uint4 y0 = lds16(at), y1 = lds16(at + 512);
      float acc[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
      const uint4* h = frags + (p * (rk >> 4) * 32 + lane) * 2;
#pragma unroll 2
      for (int kb = 0; kb < rk >> 4; ++kb) {
        const uint4 hv = h[kb * 64], lv = h[kb * 64 + 1];
        const uint32_t hi[4] = {hv.x, hv.y, hv.z, hv.w}, lo[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
          const uint4 w = lds16(at + 1024 + (kb * 2 + (t >> 1)) * 512);
          frag::mma(acc[t], hi, w.x, w.y);
          frag::mma(acc[t], lo, w.x, w.y);
          frag::mma(acc[t + 1], hi, w.z, w.w);
          frag::mma(acc[t + 1], lo, w.z, w.w);
        }
      }
      issue(b + depth * kWarps, s);
      s = s + 1 == depth ? 0 : s + 1;
      auto finish = [&](const uint4& v, int row, int half) {
        const uint32_t in_words[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 yv = frag::unpack2(in_words[t]);
          const __nv_bfloat162 r = __floats2bfloat162_rn(fmaf(scale, acc[t][half * 2], yv.x), fmaf(scale, acc[t][half * 2 + 1], yv.y));
          o[t] = *reinterpret_cast<const uint32_t*>(&r);
        }
        *reinterpret_cast<uint4*>(out + static_cast<size_t>(row) * a.ld_out + fl) = make_uint4(o[0], o[1], o[2], o[3]);
      };
      if (in && on0) finish(y0, r0, 0);
      if (in && on1) finish(y1, r1, 1);
    }
    __syncwarp();                                    // the next item's stages lie otherwise
  }
  if (!met) cg::this_cluster().barrier_wait(std::move(started));
}

template <int kTiles>
static int launch(const XpLoraArgs& a, int ranks, cudaStream_t s) {
  const int smem = smem_bytes(a.parts * a.rank, ranks, region_bytes<kTiles>());
  static std::atomic<uint64_t> allowed{0};           // devices on which the kernel may have the shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -21;
  if ((allowed >> (dev & 63) & 1) == 0) {
    if (cudaFuncSetAttribute(lora_kernel<kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kTiles * 64, kMaxCluster, region_bytes<kTiles>())) != cudaSuccess) return -21;
    allowed |= 1ull << (dev & 63);
  }
  const int most = 148 * 4 / ranks;
  pdl::launch(lora_kernel<kTiles>, static_cast<unsigned>((a.max_items < most ? a.max_items : most) * ranks), kThreads, smem, s, ranks, a, ranks);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}

}  // namespace lora
}  // namespace xpool

extern "C" int xp_lora(const XpLoraArgs* a, void* stream) {
  using namespace xpool::lora;
  if (a->rows <= 0 || a->max_items <= 0) return 0;
  if (a->parts < 1 || a->parts > XP_LORA_PARTS || a->rank < 16 || a->rank > kMaxRank || a->rank % 16 != 0 || a->k <= 0 || a->k % 8 != 0 || a->n <= 0) return -10;
  for (int p = 0; p < a->parts; ++p)
    if (a->part_end[p] % 8 != 0 || a->part_end[p] <= (p ? a->part_end[p - 1] : 0)) return -11;
  if (a->part_end[a->parts - 1] != a->n) return -11;
  auto odd = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (odd(a->x) || odd(a->y) || odd(a->out) || odd(a->a) || odd(a->b) || (a->rows > 1 && (a->ldx % 8 != 0 || a->ld_y % 8 != 0 || a->ld_out % 8 != 0))) return -12;
  // Clusters as large as the SMs hold beside one another: two CTAs to an SM, one where h has more than 256 columns. us with 1 / 2 / 4 /
  // 8 CTAs an item: 4 items of rank 16 beside 1024 -> 4096 16 / 12 / 9 / 8; 39 items of ranks 8 to 64 beside 4096 -> 6144
  // 58 / 35 / 26 / 22; 126 items beside 4096 -> 4096 of ranks 16 and 32 28 / 20 / 23 / 35, of rank 128 55 / 45 / 52 / 58, and in three
  // parts of rank 128 97 / 107 / 105 / 148.
  const int crowd = a->parts * a->rank <= 256 ? a->max_items : 2 * a->max_items;
  int ranks = crowd <= 48 ? 8 : crowd <= 80 ? 4 : crowd <= 148 ? 2 : 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->parts * a->rank <= 256 ? launch<4>(*a, ranks, s) : launch<8>(*a, ranks, s);
}
