// Attention of a chunk of new tokens over a paged KV cache.
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t.k_j - m_t),  c = scale log2(e),
//
// over the cache rows j up to the token's own; m_t is the running maximum.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int D = 128;

// One query row by a warp: lane l owns dims 4l .. 4l+3.
template <typename T, bool Q8>
__device__ __forceinline__ void attend_row(const PagedView& p, int b, int g, int len, const T* __restrict__ q,
                                           float c, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = Act<T>::to_f32(q[4 * lane + i]);
  for (int j = 0; j < len; ++j) {
    const int64_t row = pool_row(p, b, g, j);
    float k[4], v[4];
    if constexpr (Q8) {
      const float ks = __ldg(p.ks + row), vs = __ldg(p.vs + row);
      const uint32_t kw = __ldg(static_cast<const uint32_t*>(p.k) + row * 32 + lane);
      const uint32_t vw = __ldg(static_cast<const uint32_t*>(p.v) + row * 32 + lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[i] = (float)(int8_t)(kw >> (8 * i)) * ks;
        v[i] = (float)(int8_t)(vw >> (8 * i)) * vs;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[i] = Act<T>::to_f32(static_cast<const T*>(p.k)[row * D + 4 * lane + i]);
        v[i] = Act<T>::to_f32(static_cast<const T*>(p.v)[row * D + 4 * lane + i]);
      }
    }
    float s = qv[0] * k[0] + qv[1] * k[1] + qv[2] * k[2] + qv[3] * k[3];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= c;
    const float mn = fmaxf(m, s);
    const float f = mn == m ? 1.f : exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + e * v[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) out[4 * lane + i] = Act<T>::from_f32(len > 0 ? o[i] / l : 0.f);
}

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
  return dt == DIAL_F16 ? attention_t<__half>(q, p, format, out, hq, c, st)
                        : attention_t<__nv_bfloat16>(q, p, format, out, hq, c, st);
}

}  // namespace dial
