// Low-rank adapters of many requests beside a shared projection: out[r] = y[r] + scale (B (A x[r])), every row with the A, B and
// scale of its own adapter. First form: a CTA per row; warps take the rank's dot products over k, threads the features.
#include "xpool/elem.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace lora {

constexpr int kThreads = 256;
constexpr int kMaxRank = 128;

__global__ void __launch_bounds__(kThreads)
lora_kernel(XpLoraArgs a) {
  pdl::wait();
  pdl::release();
  __shared__ float h[XP_LORA_PARTS * kMaxRank];
  __shared__ int mine[2];
  if (threadIdx.x == 0) mine[0] = -2;
  __syncthreads();
  for (int i = threadIdx.x; i < min(*a.n_items, a.max_items); i += kThreads) {
    const XpLoraItem it = a.items[i];
    if (static_cast<int>(blockIdx.x) >= it.first && static_cast<int>(blockIdx.x) < it.first + it.rows) mine[0] = it.slot;
  }
  __syncthreads();
  const int slot = mine[0];
  const int r = a.perm[blockIdx.x];
  if (slot < -1 || slot >= a.slots || r < 0 || r >= a.rows) return;
  using bf16 = __nv_bfloat16;
  const bf16* x = reinterpret_cast<const bf16*>(a.x) + static_cast<size_t>(r) * a.ldx;
  const bf16* y = reinterpret_cast<const bf16*>(a.y) + static_cast<size_t>(r) * a.ld_y;
  bf16* out = reinterpret_cast<bf16*>(a.out) + static_cast<size_t>(r) * a.ld_out;
  const int rank = slot >= 0 ? a.ranks[slot] : 0;
  const float scale = slot >= 0 ? a.scale[slot] : 0.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int j = warp; j < a.parts * rank; j += kThreads / 32) {
    const bf16* row = reinterpret_cast<const bf16*>(a.a) + ((static_cast<size_t>(slot) * a.parts + j / rank) * a.rank + j % rank) * a.k;
    float s = 0.f;
    for (int c = lane; c < a.k; c += 32) s += elem::ld(x + c) * elem::ld(row + c);
    s = elem::warp_sum(s);
    if (lane == 0) h[j] = s;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.n; c += kThreads) {
    int part = 0;
    while (c >= a.part_end[part]) ++part;
    const bf16* row = reinterpret_cast<const bf16*>(a.b) + (static_cast<size_t>(max(slot, 0)) * a.n + c) * a.rank;
    float s = 0.f;
    for (int j = 0; j < rank; ++j) s += h[part * rank + j] * elem::ld(row + j);
    elem::st(out + c, elem::ld(y + c) + scale * s);
  }
}

}  // namespace lora
}  // namespace xpool

extern "C" int xp_lora(const XpLoraArgs* a, void* stream) {
  using namespace xpool::lora;
  if (a->rows <= 0) return 0;
  if (a->parts < 1 || a->parts > XP_LORA_PARTS || a->rank < 16 || a->rank > kMaxRank || a->rank % 16 != 0 || a->k <= 0 || a->n <= 0) return -10;
  if (a->part_end[a->parts - 1] != a->n) return -11;
  xpool::pdl::launch(lora_kernel, a->rows, kThreads, 0, reinterpret_cast<cudaStream_t>(stream), 1, *a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}
