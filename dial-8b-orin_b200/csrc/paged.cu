// Paged KV caches: the post-QKV step that writes pages, and reading them back.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int D = 128;

// Eight values as four pairs.
template <typename T>
__device__ __forceinline__ void unpack8(uint4 u, float2 (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float2 (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __float22half2_rn(v[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Row scale and reciprocal of the int8 rows: absmax / 127, 1 for rows without
// a usable absmax (below 1e-30, where scales and reciprocals near the ends of
// f32's range: the codes are zeros, off by less than 1e-30).
__device__ __forceinline__ void row_scale(float amax, float& s, float& inv) {
  s = amax >= 1e-30f ? __fdiv_rn(amax, 127.0f) : 1.0f;
  inv = __fdiv_rn(1.0f, s);
}
// round(x / s), halves away from zero, clamped to +-127
__device__ __forceinline__ uint32_t code(float x, float inv) {
  const float r = fminf(fmaxf(roundf(__fmul_rn(x, inv)), -127.f), 127.f);
  return (uint32_t)(int)r & 0xFFu;
}

// ------------------------------------------------------------------ append
// Eight lanes per head: lane j holds elements 8j .. 8j+7 and 64+8j .. 64+8j+7, so the
// pairs (i, i + 64) stay in the lane, and four heads share a warp's look-ups, shuffles and
// reciprocal root.  `wpt` warps share a token: each looks up the page row and the token's
// cosines, then walks heads, the next ones' values on their way while it works on four.
// Few tokens: a head per eight lanes once; many: as few warps a token as fill the SMs, as
// the look-ups cost about what four heads do.  2048 tokens of 32 + 2 * 8 heads in bf16 take
// 15.5 us (50 MB, 3.2 TB/s), twice what the bytes need; bound by the chain of a head's steps
// (sum, exchange, root, turn, pack) over two CTAs an SM: issue 40 %, and two or three heads
// on their way instead of one change nothing.  A warp per head took 28.6 us, a warp per
// token with two heads in it 15.8.
// The mean square is summed in f64 (its squares are exact there) and 1/sqrt refined by one
// Newton step in f64, so that the f32 factor -- and with it every int8 code -- does not
// depend on the order of a sum; each later product is rounded to f32 on its own for the
// same reason.
template <typename T, bool Q8>
__global__ void __launch_bounds__(256)
    paged_append_kernel(const T* __restrict__ qkv, RopeArgs r, PagedView p, T* __restrict__ q_out, int hq, int wpt) {
  pdl_begin();
  const int64_t w = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5), t = w / wpt;
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) chunk_of(p, b, true);
  if (t >= p.tokens) return;
  const int heads = hq + 2 * p.hkv, step = 4 * wpt;
  const int j = threadIdx.x & 7;
  const unsigned part = 0xFFu << (threadIdx.x & 24);
  int h = (int)(w - t * wpt) * 4 + ((threadIdx.x >> 3) & 3);
  const T* tok = qkv + (t * heads + h) * D + 8 * j;  // this lane's first values of head h
  uint4 na = make_uint4(0, 0, 0, 0), nz = na;
  if (h < heads) {
    na = __ldg(reinterpret_cast<const uint4*>(tok));
    nz = __ldg(reinterpret_cast<const uint4*>(tok + 64));
  }
  const int b = seq_of_token(p.q_start, p.n_seqs, t);
  if (b >= p.n_seqs) return;  // behind the last sequence
  const Chunk c = chunk_of(p, b, false);
  if (t < c.q0 || t >= c.q0 + c.n) return;
  // the token's turns
  float2 cs[4], sn[4];
  {
    const uint32_t axes = r.axis[j >> 1] >> (16 * (j & 1));
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
      const float4* x = reinterpret_cast<const float4*>(r.cos_t + (int64_t)row[0] * (D / 2) + 8 * j);
      const float4* y = reinterpret_cast<const float4*>(r.sin_t + (int64_t)row[0] * (D / 2) + 8 * j);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 u = __ldg(x + i), v = __ldg(y + i);
        cs[2 * i] = make_float2(u.x, u.y), cs[2 * i + 1] = make_float2(u.z, u.w);
        sn[2 * i] = make_float2(v.x, v.y), sn[2 * i + 1] = make_float2(v.z, v.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int ax = (axes >> (2 * i)) & 3;
        const int64_t at = (int64_t)(ax == 0 ? row[0] : ax == 1 ? row[1] : ax == 2 ? row[2] : row[3]) * (D / 2) + 8 * j + i;
        const float u = __ldg(r.cos_t + at), v = __ldg(r.sin_t + at);
        if (i & 1) cs[i / 2].y = u, sn[i / 2].y = v;
        else cs[i / 2].x = u, sn[i / 2].x = v;
      }
    }
  }
  // the token's row of its page, for kv head 0 (heads are a page's rows apart)
  const int at = c.kv - c.n + (int)(t - c.q0);
  int64_t row0 = -1;
  if (at >= 0) {
    const int page = __ldg(p.table + (int64_t)b * p.max_pages + (at >> p.log2_page));
    if (page < 0 || page >= p.n_pages) {
      flag_invalid(p.err);
    } else {
      row0 = (((int64_t)page * p.hkv) << p.log2_page) + (at & ((1 << p.log2_page) - 1));
    }
  }
  float2 wa[4] = {}, wz[4] = {};  // norm weights of the heads at hand: q's, then k's
  int kind = 0;
  T* qdst = q_out + (t * hq + h) * D + 8 * j;
  for (; h < heads; h += step, tok += step * D, qdst += step * D) {
    float2 a[4], z[4];
    unpack8<T>(na, a);
    unpack8<T>(nz, z);
    if (h + step < heads) {
      na = __ldg(reinterpret_cast<const uint4*>(tok + step * D));
      nz = __ldg(reinterpret_cast<const uint4*>(tok + step * D + 64));
    }
    if (h < hq + p.hkv) {
      if (r.qn) {
        const int now = h < hq ? 1 : 2;
        if (now != kind) {
          const T* wt = static_cast<const T*>(h < hq ? r.qn : r.kn) + 8 * j;
          unpack8<T>(__ldg(reinterpret_cast<const uint4*>(wt)), wa);
          unpack8<T>(__ldg(reinterpret_cast<const uint4*>(wt + 64)), wz);
          kind = now;
        }
        double ss = 0.0, s2 = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double x = a[i].x, y = a[i].y, u = z[i].x, v = z[i].y;
          ss = fma(x, x, ss), s2 = fma(u, u, s2);
          ss = fma(y, y, ss), s2 = fma(v, v, s2);
        }
        ss += s2;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(part, ss, o);
        const double m = fma(ss, 1.0 / D, (double)r.eps);
        const float mf = (float)m;
        double y;
        if (mf > 1e-30f && mf < 1e30f) {
          y = (double)rsqrtf(mf);
          y = y * fma(-0.5 * m * y, y, 1.5);
        } else {
          y = 1.0 / sqrt(m);
        }
        const float inv = (float)y;
        const float2 iv = make_float2(inv, inv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = mul2(mul2(a[i], iv), wa[i]);
          z[i] = mul2(mul2(z[i], iv), wz[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = a[i], y = z[i];
        a[i].x = __fsub_rn(__fmul_rn(x.x, cs[i].x), __fmul_rn(y.x, sn[i].x));
        a[i].y = __fsub_rn(__fmul_rn(x.y, cs[i].y), __fmul_rn(y.y, sn[i].y));
        z[i].x = __fadd_rn(__fmul_rn(x.x, sn[i].x), __fmul_rn(y.x, cs[i].x));
        z[i].y = __fadd_rn(__fmul_rn(x.y, sn[i].y), __fmul_rn(y.y, cs[i].y));
      }
      if (h < hq) {
        *reinterpret_cast<uint4*>(qdst) = pack8<T>(a);
        *reinterpret_cast<uint4*>(qdst + 64) = pack8<T>(z);
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
        const float v[4] = {a[i].x, a[i].y, z[i].x, z[i].y};
#pragma unroll
        for (int x = 0; x < 4; ++x) amax = fmaxf(amax, fabsf(v[x])), odd |= !(fabsf(v[x]) < INFINITY);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(part, amax, o));
      odd = __any_sync(part, odd);
      float s, inv;
      row_scale(amax, s, inv);
      uint2 lo = make_uint2(0, 0), hi = lo;
      if (odd) {
        s = __int_as_float(0x7fc00000);  // a row with a NaN or an infinity is kept as NaN
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = (code(a[i].x, inv) | code(a[i].y, inv) << 8) << (16 * (i & 1));
          const uint32_t y = (code(z[i].x, inv) | code(z[i].y, inv) << 8) << (16 * (i & 1));
          if (i < 2) lo.x |= x, hi.x |= y;
          else lo.y |= x, hi.y |= y;
        }
      }
      int8_t* dst = static_cast<int8_t*>(const_cast<void*>(is_k ? p.k : p.v)) + row * D + 8 * j;
      *reinterpret_cast<uint2*>(dst) = lo;
      *reinterpret_cast<uint2*>(dst + 64) = hi;
      if (j == 0) const_cast<float*>(is_k ? p.ks : p.vs)[row] = s;
    } else {
      T* dst = static_cast<T*>(const_cast<void*>(is_k ? p.k : p.v)) + row * D + 8 * j;
      *reinterpret_cast<uint4*>(dst) = pack8<T>(a);
      *reinterpret_cast<uint4*>(dst + 64) = pack8<T>(z);
    }
  }
}

// ------------------------------------------------------------------ read
// A warp per token: its page row is looked up once, then its 2 Hkv rows (keys first) go by
// two at a time, 8 values a lane, four rounds of loads in flight.  Bound by the bytes:
// 64K rows of 8 int8 heads take 38 us, 5.4 TB/s.
template <typename T, bool Q8>
__global__ void __launch_bounds__(256)
    paged_read_kernel(PagedView p, T* __restrict__ k_out, T* __restrict__ v_out) {
  pdl_begin();
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.n_seqs; b += blockDim.x) chunk_of(p, b, true);
  const int64_t t = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int b = seq_of_token(p.q_start, p.n_seqs, t);
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
  const int most = (hq + 2 * p.hkv + 3) / 4;  // eight lanes per head
  const int wpt = (int)std::min<int64_t>(most, std::max<int64_t>(1, 16 * (int64_t)sm_count() / p.tokens));
  const int64_t blocks = (p.tokens * wpt + 7) / 8;
  if (blocks >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many tokens (%lld)", (long long)p.tokens);
  const dim3 grid((unsigned)blocks);
  auto k = format == DIAL_KV_INT8 ? paged_append_kernel<T, true> : paged_append_kernel<T, false>;
  return launch_pdl("paged_append_kernel", k, grid, dim3(256), 0, st, static_cast<const T*>(qkv), r, p,
                    static_cast<T*>(q_out), hq, wpt);
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
