// Attention over a paged KV cache: the row-by-row form, and the launchers of the others.
#pragma once

#include <type_traits>

#include "paged.cuh"
#include "tma.cuh"

namespace dial {
namespace pa {

// Bounded wait that other kinds of errors in the flag do not cut short.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int* err) {
  if (tma::mbar_try(bar, parity)) return true;
  const unsigned long long t0 = tma::global_ns();
  for (uint32_t i = 1;; ++i) {
    if (tma::mbar_try(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*(volatile int*)err == (int)DIAL_ERR_TIMEOUT) return false;
      if (tma::global_ns() - t0 > tma::kWaitNs) {
        atomicExch(err, (int)DIAL_ERR_TIMEOUT);
        return false;
      }
    }
  }
}
// P is rounded once, to the 16 bits that the matrix instructions take; its sum is of the
// unrounded values.  P = 2^(s - m) with m kLift below a maximum of the row, which moves when a
// score passes it by kGrow more: f16 operands (and int8 pages, whose P carries the value's
// scale) have P in [0, 2^15], so that a weight of 2^-21 of the row's largest still has its 11
// bits and the last bit is 2^-31 of it.  From 1 instead of 2^7 on, 2048 keys 22 octaves below a
// first one without a value were off by 2^-9.4 of their sum.  bf16's range needs no lift.
constexpr float kGrow = 8.f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;
// Whether a row's sum l, in units of its maximum m, came about in P's range.  Over 16-bit pages
// m is a rounded product, c S, and P = 2^(c S - m) an exact difference: below 2^23 they agree to
// half an octave, so that the row's largest P is 2^(LIFT - 1/2) or more.  Scores far above that
// leave it anywhere, and a row whose largest P came out small is computed again.
template <typename T>
__device__ __forceinline__ bool in_range(float l, float m) {
  return l >= (kLift<T> > 0.f ? 64.f : 0.5f) || m == -INFINITY;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float4 lds16f(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// int8x4 -> two 16-bit pairs, exact.  f16: 1024 + (b + 128) by a byte permute, less
// 1152.  bf16: 128 + (b & 127) less 128 or 256 by the sign bit.
template <typename T>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi);
template <>
__device__ __forceinline__ void widen<__half>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u, bias = 0x64806480u;
  const uint32_t a = prmt(u, 0x64646464u, 0x4140u), b = prmt(u, 0x64646464u, 0x4342u);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
template <>
__device__ __forceinline__ void widen<__nv_bfloat16>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t tl = prmt(w, 0x43434343u, 0x4140u), th = prmt(w, 0x43434343u, 0x4342u);
  const uint32_t l1 = tl & 0xFF7FFF7Fu, l2 = (tl & 0x00800080u) | 0x43004300u;
  const uint32_t h1 = th & 0xFF7FFF7Fu, h2 = (th & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&l1), *reinterpret_cast<const __nv_bfloat162*>(&l2));
  const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&h1), *reinterpret_cast<const __nv_bfloat162*>(&h2));
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster16(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

}  // namespace pa

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
    const float f = mn == m ? 1.f : exp2f(m - mn), e = s == -INFINITY ? 0.f : exp2f(s - mn);
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
