// Attention over a paged KV cache: the row-by-row form, and the launchers of the others.
#pragma once

#include "paged.cuh"

namespace dial {

// One query row by a warp: lane l owns dims 4l .. 4l+3.
template <typename T, bool Q8>
__device__ __noinline__ void attend_row(const PagedView& p, int b, int g, int len, const T* __restrict__ q,
                                           float c, T* __restrict__ out) {
  constexpr int D = 128;
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

dial_status launch_paged_attention_tiles(const void* q, const PagedView& p, int format, void* out, dial_dtype dt,
                                         int hq, int64_t max_kv, float c, cudaStream_t st);

}  // namespace dial
