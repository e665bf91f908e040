// Attention of query rows over a prefix that they share: the pieces of a plan (a range of a prefix, and the consecutive rows that
// read it) leave partial results, un-normalised sums with their maximum and sum of weights, to which the decode kernel adds the
// tokens of each row's own. First form: four lanes hold a query head, every token is read from global memory.
#include <math_constants.h>

#include "xpool/elem.cuh"
#include "xpool/pdl.cuh"
#include "xpool/request_api.h"

namespace xpool {
namespace prefix {

constexpr int kThreads = 128;

template <int D>
__global__ void __launch_bounds__(kThreads)
shared_prefix_kernel(XpDecodeSharedArgs args) {
  pdl::wait();
  pdl::release();
  const XpDecodeAttnArgs& a = args.a;
  if (static_cast<int>(blockIdx.x) >= min(*args.n_pieces, args.max_pieces)) return;
  const XpPrefixPiece p = args.pieces[blockIdx.x];
  const int hk = blockIdx.y, G = a.q_heads / a.kv_heads;
  const int slots = args.max_parts + (a.num_splits > 1 ? a.num_splits : 0);
  const int quad = threadIdx.x >> 2, part = threadIdx.x & 3;
  constexpr int E = D / 4;
  const int page_shift = 31 - __clz(a.page_size);
  const int* table = a.block_table + static_cast<size_t>(p.leader) * a.max_blocks;
  for (int base = 0; base < p.rows * G; base += kThreads / 4) {
    const int i = base + quad;
    const bool on = i < p.rows * G;
    const int row = p.row0 + (on ? i / G : 0), hq = hk * G + (on ? i % G : 0);
    const __nv_bfloat16* qp = reinterpret_cast<const __nv_bfloat16*>(a.q) + (static_cast<size_t>(row) * a.q_heads + hq) * D + part * E;
    float q[E], acc[E], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = elem::ld(qp + e) * a.scale * 1.4426950408889634f, acc[e] = 0.f;
    for (int t = p.tok0; t < p.tok1; ++t) {
      const int page = min(max(table[t >> page_shift], 0), a.num_pages - 1);
      const size_t tok = (static_cast<size_t>(page) << page_shift) + (t & (a.page_size - 1));
      const __nv_bfloat16* k = reinterpret_cast<const __nv_bfloat16*>(a.k_cache) + (tok * a.kv_heads + hk) * D + part * E;
      const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v_cache) + (tok * a.kv_heads + hk) * D + part * E;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += q[e] * elem::ld(k + e);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      const float top = fmaxf(m, s), c = exp2f(m - top), w = exp2f(s - top);
      m = top, l = l * c + w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + w * elem::ld(v + e);
    }
    if (!on) continue;
    const size_t at = (static_cast<size_t>(row) * a.q_heads + hq) * slots + p.part;
#pragma unroll
    for (int e = 0; e < E; ++e) a.ws[at * D + part * E + e] = acc[e];
    if (part == 0) {
      float* ml = a.ws + static_cast<size_t>(a.batch) * a.q_heads * slots * D + at * 2;
      ml[0] = m, ml[1] = l;
    }
  }
}

}  // namespace prefix
}  // namespace xpool

extern "C" int xp_shared_prefix_pieces(const XpDecodeSharedArgs* r, void* stream) {
  using namespace xpool::prefix;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(r->max_pieces, r->a.kv_heads);
  if (r->a.head_dim == 128) xpool::pdl::launch(shared_prefix_kernel<128>, grid, kThreads, 0, s, 1, *r);
  else xpool::pdl::launch(shared_prefix_kernel<64>, grid, kThreads, 0, s, 1, *r);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - static_cast<int>(e);
}
