// Attention of a chunk of new tokens over a paged KV cache.
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t.k_j - m_t),  c = scale log2(e),
//
// over the cache rows j up to the token's own; m_t is the running maximum.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"

namespace dial {

namespace {

constexpr int D = 128;

// A warp per (token, query head).
template <typename T, bool Q8>
__global__ void __launch_bounds__(128)
    paged_attention_rows_kernel(const T* __restrict__ q, PagedView p, T* __restrict__ out, int hq, float c) {
  pdl_begin();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) chunk_of(p, b, true);
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int b = seq_of_token(p, t);
  if (b >= p.n_seqs || h >= hq) return;
  const Chunk ch = chunk_of(p, b, false);
  if (t < ch.q0 || t >= ch.q0 + ch.n) return;
  const int len = ch.kv - ch.n + (int)(t - ch.q0) + 1;
  attend_row<T, Q8>(p, b, h / (hq / p.hkv), len, q + (t * hq + h) * D, c, out + (t * hq + h) * D);
}

}  // namespace

template <typename T>
static dial_status attention_t(const void* q, const PagedView& p, int format, void* out, int hq, float c,
                               cudaStream_t st) {
  const dim3 grid((unsigned)p.tokens, (unsigned)((hq + 3) / 4));
  auto k = format == DIAL_KV_INT8 ? paged_attention_rows_kernel<T, true> : paged_attention_rows_kernel<T, false>;
  return launch_pdl("paged_attention_rows_kernel", k, grid, dim3(128), 0, st, static_cast<const T*>(q), p,
                    static_cast<T*>(out), hq, c);
}

dial_status launch_paged_attention(const void* q, const PagedView& p, int format, void* out, dial_dtype dt,
                                   int hq, int64_t max_kv, float scale, cudaStream_t st) {
  const float c = (float)((double)scale * 1.4426950408889634);
  if (max_kv > 0) return launch_paged_attention_tiles(q, p, format, out, dt, hq, max_kv, c, st);
  return dt == DIAL_F16 ? attention_t<__half>(q, p, format, out, hq, c, st)
                        : attention_t<__nv_bfloat16>(q, p, format, out, hq, c, st);
}

}  // namespace dial
