// Paged KV caches: the post-QKV step that writes pages, and reading them back.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int D = 128;

template <typename T>
__device__ __forceinline__ void unpack4(uint2 u, float (&v)[4]) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Act<T>::to_f32(h[i]);
}
template <typename T>
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) {
  uint2 u;
  T* h = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = Act<T>::from_f32(v[i]);
  return u;
}

// Row scale and reciprocal of the int8 rows: absmax / 127, 1 for rows without
// a usable absmax (below 1e-36 its reciprocal would overflow: the codes are
// zeros, off by less than 1e-36).
__device__ __forceinline__ void row_scale(float amax, float& s, float& inv) {
  s = amax >= 1e-36f ? __fdiv_rn(amax, 127.0f) : 1.0f;
  inv = __fdiv_rn(1.0f, s);
}
// round(x / s), halves away from zero, clamped to +-127
__device__ __forceinline__ uint32_t code(float x, float inv) {
  const float r = fminf(fmaxf(roundf(__fmul_rn(x, inv)), -127.f), 127.f);
  return (uint32_t)(int)r & 0xFFu;
}

// ------------------------------------------------------------------ append
// A half-warp per head: lane j of 16 holds elements 4j .. 4j+3 and 64+4j .. 64+4j+3, so
// the pairs (i, i + 64) stay in the lane.  A CTA is one token (or a part of its heads): the
// page row and the token's cosines are looked up once and every half-warp walks heads, the
// next one's values on their way while it works on one.  Bound by the bytes of qkv, q and
// the cache rows.
// The mean square is summed in f64 (its squares are exact there) and 1/sqrt refined by one
// Newton step in f64, so that the f32 factor -- and with it every int8 code -- does not
// depend on the order of a sum; each later product is rounded to f32 on its own for the
// same reason.
template <typename T, bool Q8>
__global__ void __launch_bounds__(256)
    paged_append_kernel(const T* __restrict__ qkv, RopeArgs r, PagedView p, T* __restrict__ q_out, int hq) {
  pdl_begin();
  const int64_t t = blockIdx.x;
  const int heads = hq + 2 * p.hkv, step = gridDim.y * 16;
  const int j = threadIdx.x & 15;
  const unsigned half = 0xFFFFu << (threadIdx.x & 16);
  int h = blockIdx.y * 16 + (threadIdx.x >> 4);
  const T* tok = qkv + t * heads * D;
  uint2 na = make_uint2(0, 0), nz = na;
  if (h < heads) {
    na = __ldg(reinterpret_cast<const uint2*>(tok + h * D) + j);
    nz = __ldg(reinterpret_cast<const uint2*>(tok + h * D + 64) + j);
  }
  if (t == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) chunk_of(p, b, true);
  const int b = seq_of_token(p, t);
  if (b >= p.n_seqs) return;  // behind the last sequence
  const Chunk c = chunk_of(p, b, false);
  if (t < c.q0 || t >= c.q0 + c.n) return;
  // the token's turns
  float cs[4], sn[4];
  {
    const uint32_t axes = r.axis[j >> 2] >> (8 * (j & 3));
    int row[4] = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x < r.n_axes) {
        int v = __ldg(r.pos + x * p.tokens + t);
        if (v < 0 || v >= r.table_rows) {
          flag_invalid(p.err);
          v = v < 0 ? 0 : (int)r.table_rows - 1;
        }
        row[x] = v;
      }
    if (r.n_axes == 1) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(r.cos_t + (int64_t)row[0] * (D / 2)) + j);
      const float4 y = __ldg(reinterpret_cast<const float4*>(r.sin_t + (int64_t)row[0] * (D / 2)) + j);
      cs[0] = x.x, cs[1] = x.y, cs[2] = x.z, cs[3] = x.w;
      sn[0] = y.x, sn[1] = y.y, sn[2] = y.z, sn[3] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ax = (axes >> (2 * i)) & 3;
        const int64_t at = (int64_t)(ax == 0 ? row[0] : ax == 1 ? row[1] : ax == 2 ? row[2] : row[3]) * (D / 2) + 4 * j + i;
        cs[i] = __ldg(r.cos_t + at), sn[i] = __ldg(r.sin_t + at);
      }
    }
  }
  // the token's row of its page, for kv head 0 (heads are a page's rows apart)
  const int at = c.kv - c.n + (int)(t - c.q0);
  int64_t row0 = -1;
  if (at >= 0) {
    const int page = __ldg(p.table + (int64_t)b * p.max_pages + (at >> p.log2_page));
    if (page < 0 || page >= p.n_pages) {
      if (threadIdx.x == 0) flag_invalid(p.err);
    } else {
      row0 = (((int64_t)page * p.hkv) << p.log2_page) + (at & ((1 << p.log2_page) - 1));
    }
  }
  for (; h < heads; h += step) {
    float a[4], z[4];
    unpack4<T>(na, a);
    unpack4<T>(nz, z);
    if (h + step < heads) {
      na = __ldg(reinterpret_cast<const uint2*>(tok + (h + step) * D) + j);
      nz = __ldg(reinterpret_cast<const uint2*>(tok + (h + step) * D + 64) + j);
    }
    if (h < hq + p.hkv) {
      const T* w = static_cast<const T*>(h < hq ? r.qn : r.kn);
      if (w) {
        float wa[4], wz[4];
        unpack4<T>(__ldg(reinterpret_cast<const uint2*>(w) + j), wa);
        unpack4<T>(__ldg(reinterpret_cast<const uint2*>(w + 64) + j), wz);
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += (double)a[i] * a[i] + (double)z[i] * z[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(half, ss, o);
        const double m = ss / D + (double)r.eps;
        double y;
        if (m > 1e-30 && m < 1e30) {
          y = (double)rsqrtf((float)m);
          y = y * (1.5 - 0.5 * m * y * y);
        } else {
          y = 1.0 / sqrt(m);
        }
        const float inv = (float)y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = __fmul_rn(__fmul_rn(a[i], inv), wa[i]);
          z[i] = __fmul_rn(__fmul_rn(z[i], inv), wz[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = a[i], y = z[i];
        a[i] = __fsub_rn(__fmul_rn(x, cs[i]), __fmul_rn(y, sn[i]));
        z[i] = __fadd_rn(__fmul_rn(x, sn[i]), __fmul_rn(y, cs[i]));
      }
      if (h < hq) {
        T* dst = q_out + (t * hq + h) * D;
        reinterpret_cast<uint2*>(dst)[j] = pack4<T>(a);
        reinterpret_cast<uint2*>(dst + 64)[j] = pack4<T>(z);
        continue;
      }
    }
    if (row0 < 0) continue;
    const bool is_k = h < hq + p.hkv;
    const int64_t row = row0 + ((int64_t)(is_k ? h - hq : h - hq - p.hkv) << p.log2_page);
    if constexpr (Q8) {
      float amax = 0.f;
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        amax = fmaxf(amax, fmaxf(fabsf(a[i]), fabsf(z[i])));
        odd |= !(fabsf(a[i]) < INFINITY) || !(fabsf(z[i]) < INFINITY);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(half, amax, o));
      odd = __any_sync(half, odd);
      float s, inv;
      row_scale(amax, s, inv);
      uint32_t lo = 0, hi = 0;
      if (odd) {
        s = __int_as_float(0x7fc00000);  // a row with a NaN or an infinity is kept as NaN
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo |= code(a[i], inv) << (8 * i);
          hi |= code(z[i], inv) << (8 * i);
        }
      }
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<int8_t*>(const_cast<void*>(is_k ? p.k : p.v)) + row * D);
      dst[j] = lo;
      dst[16 + j] = hi;
      if (j == 0) const_cast<float*>(is_k ? p.ks : p.vs)[row] = s;
    } else {
      T* dst = static_cast<T*>(const_cast<void*>(is_k ? p.k : p.v)) + row * D;
      reinterpret_cast<uint2*>(dst)[j] = pack4<T>(a);
      reinterpret_cast<uint2*>(dst + 64)[j] = pack4<T>(z);
    }
  }
}

// ------------------------------------------------------------------ read
// A warp per token: its page row is looked up once, then its 2 Hkv rows (keys first) go by
// two at a time, 8 values a lane, four rounds of loads in flight.  Bound by the bytes.
template <typename T, bool Q8>
__global__ void __launch_bounds__(256)
    paged_read_kernel(PagedView p, T* __restrict__ k_out, T* __restrict__ v_out) {
  pdl_begin();
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) chunk_of(p, b, true);
  const int64_t t = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int b = seq_of_token(p, t);
  if (b >= p.n_seqs) return;
  const Chunk c = chunk_of(p, b, false);
  if (t < c.q0 || t >= c.q0 + c.n) return;
  const int h0 = (threadIdx.x >> 4) & 1, j = threadIdx.x & 15;
  const int at = c.kv - c.n + (int)(t - c.q0);
  const int64_t row0 = at >= 0 ? pool_row(p, b, 0, at) : -1;
  constexpr int U = 4;
  for (int i0 = 0; i0 < p.hkv; i0 += U) {
    uint4 o[U];
    float sc[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = 2 * (i0 + i) + h0;
      o[i] = make_uint4(0, 0, 0, 0);
      sc[i] = 0.f;
      if (h >= 2 * p.hkv || row0 < 0) continue;
      const bool is_k = h < p.hkv;
      const int64_t row = row0 + ((int64_t)(is_k ? h : h - p.hkv) << p.log2_page);
      const void* src = is_k ? p.k : p.v;
      if constexpr (Q8) {
        sc[i] = __ldg((is_k ? p.ks : p.vs) + row);
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(static_cast<const int8_t*>(src) + row * D) + j);
        o[i].x = q.x, o[i].y = q.y;
      } else {
        o[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(src) + row * D) + j);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int h = 2 * (i0 + i) + h0;
      if (h >= 2 * p.hkv) continue;
      const bool is_k = h < p.hkv;
      if constexpr (Q8) {
        const uint2 q = make_uint2(o[i].x, o[i].y);
        T* e = reinterpret_cast<T*>(&o[i]);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          e[x] = Act<T>::from_f32((float)(int8_t)((x < 4 ? q.x : q.y) >> (8 * (x & 3))) * sc[i]);
      }
      T* dst = (is_k ? k_out : v_out) + (t * p.hkv + (is_k ? h : h - p.hkv)) * D + 8 * j;
      *reinterpret_cast<uint4*>(dst) = o[i];
    }
  }
}

}  // namespace

template <typename T>
static dial_status append_t(const void* qkv, const RopeArgs& r, const PagedView& p, int format, void* q_out,
                            int hq, cudaStream_t st) {
  // few tokens: 16 heads a CTA, for latency; otherwise a CTA per token
  const dim3 grid((unsigned)p.tokens, p.tokens < 2 * sm_count() ? (unsigned)((hq + 2 * p.hkv + 15) / 16) : 1u);
  auto k = format == DIAL_KV_INT8 ? paged_append_kernel<T, true> : paged_append_kernel<T, false>;
  return launch_pdl("paged_append_kernel", k, grid, dim3(256), 0, st, static_cast<const T*>(qkv), r, p,
                    static_cast<T*>(q_out), hq);
}

dial_status launch_paged_append(const void* qkv, const RopeArgs& r, const PagedView& p, int format,
                                void* q_out, dial_dtype dt, int hq, cudaStream_t st) {
  return dt == DIAL_F16 ? append_t<__half>(qkv, r, p, format, q_out, hq, st)
                        : append_t<__nv_bfloat16>(qkv, r, p, format, q_out, hq, st);
}

template <typename T>
static dial_status read_t(const PagedView& p, int format, void* k_out, void* v_out, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.tokens + 7) / 8);
  auto k = format == DIAL_KV_INT8 ? paged_read_kernel<T, true> : paged_read_kernel<T, false>;
  return launch_pdl("paged_read_kernel", k, dim3(grid), dim3(256), 0, st, p, static_cast<T*>(k_out),
                    static_cast<T*>(v_out));
}

dial_status launch_paged_read(const PagedView& p, int format, void* k_out, void* v_out, dial_dtype dt,
                              cudaStream_t st) {
  return dt == DIAL_F16 ? read_t<__half>(p, format, k_out, v_out, st)
                        : read_t<__nv_bfloat16>(p, format, k_out, v_out, st);
}

}  // namespace dial
