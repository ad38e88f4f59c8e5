// Attention over a paged KV cache for few query rows (decoding, drafted tokens):
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t.k_j - m_t),  c = scale log2(e),
//
// over the cache rows j up to the token's own.  The rows of a sequence and kv head
// (token x query head of the group, at most 32) share every key, so the work is
// bound by the bytes of the cache.
//
// A CTA takes a share of the key tiles of one (sequence, kv head); its four warps
// take tiles in turn, each through a ring of its own of three 8 KB stages that one
// lane fills by TMA (SWIZZLE_128B boxes of at most 16 or 32 rows of a page) -- 192 KB
// in flight on an SM with its two CTAs.  Scores and P V run on mma.sync m16n8k16,
// which these few rows do not need more of.
//   16-bit pages: 16 keys a tile, operands by ldmatrix (V transposed).
//   int8 pages: 32 keys a tile, widened in registers.  The order of the 128 dims in
//   Q K^T is free as long as Q follows it: a lane takes 16 consecutive bytes of a key,
//   so two 16-byte loads a key feed 8 k-steps; V's 4 x 4 byte blocks are transposed
//   with byte permutes, and the dims of O come out permuted.  Scales as in
//   paged_attention_tiles.cu: k_s on the score, log2 v_s in the exponent, 1 / v_s in
//   the row sum.
// The warps' (m, l, O) meet in shared memory, the CTAs' in the cluster's: no
// workspace, no counters, and the same result whatever the timing.
#include <cuda.h>

#include <algorithm>

#include "paged.cuh"
#include "paged_attention.cuh"
#include "tma.cuh"

namespace dial {

namespace {

using namespace pa;
using namespace tma;

constexpr int D = 128;
constexpr int WARPS = 4;
constexpr int STAGES = 3;
constexpr int TILE = 4096;            // bytes of a K or V tile
constexpr int STAGE = 2 * TILE;
constexpr int RING = WARPS * STAGES * STAGE;

struct Args {
  PagedView p;
  int hq, rep;
  float c;
  const void* q;
  void* out;
};

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster16(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// MT: 16-row tiles of query rows (rows of the chunk = token * rep + head)
template <typename T, bool Q8, int MT>
__global__ void __launch_bounds__(WARPS * 32, 2)
    paged_attention_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                const Args a) {
  constexpr int TK = Q8 ? 32 : 16;  // keys per tile
  constexpr int NT = TK / 8;        // 8-key column tiles of the scores
  constexpr int ROWS = 16 * MT;
  using PT = typename std::conditional<Q8, __half, T>::type;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float sm_m[WARPS][ROWS], sm_l[WARPS][ROWS], cta_m[ROWS], cta_l[ROWS];
  __shared__ __align__(8) uint64_t bars[WARPS * STAGES];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, qd = lane & 3;
  int* err = a.p.err;
  pdl_trigger();
  const uint32_t bar = smem_u32(&bars[warp * STAGES]), ring = base + warp * STAGES * STAGE;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bar + 8 * s, 1);
    fence_barrier_init();
    fence_proxy_async();
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  __syncwarp();
  pdl_wait();

  const int S = (int)cluster_size(), rank = (int)cluster_rank();
  const int unit = blockIdx.x / S, b = unit / a.p.hkv, g = unit % a.p.hkv;
  const Chunk ch = chunk_of(a.p, b, threadIdx.x == 0);
  const int before = ch.kv - ch.n;                     // token i sees keys 0 .. before + i
  const int len = ch.n > 0 ? ch.kv : 0;
  const int ntile = (len + TK - 1) / TK;
  const int t0 = (int)((int64_t)ntile * rank / S), t1 = (int)((int64_t)ntile * (rank + 1) / S);
  const int page = 1 << a.p.log2_page;

  auto fetch = [&](int tile, int st) {  // by lane 0
    const int k0 = tile * TK;
    const uint32_t dst = ring + st * STAGE, fb = bar + 8 * st;
    if constexpr (Q8) {
      const int box = min(page, TK), n = min(TK / box, (ch.kv - k0 + box - 1) / box);
      mbar_expect_tx(fb, (uint32_t)(2 * n * box * 128));
      for (int x = 0; x < n; ++x) {
        const int row = (int)pool_row(a.p, b, g, k0 + x * box);
        load_2d(dst + x * box * 128, &kmap, fb, 0, row);
        load_2d(dst + TILE + x * box * 128, &vmap, fb, 0, row);
      }
    } else {
      const int row = (int)pool_row(a.p, b, g, k0);
      mbar_expect_tx(fb, STAGE);
      load_2d(dst, &kmap, fb, 0, row);
      load_2d(dst + TILE / 2, &kmap, fb, 128, row);
      load_2d(dst + TILE, &vmap, fb, 0, row);
      load_2d(dst + TILE + TILE / 2, &vmap, fb, 128, row);
    }
  };
  if (lane == 0)
    for (int s = 0; s < STAGES; ++s)
      if (t0 + warp + s * WARPS < t1) fetch(t0 + warp + s * WARPS, s);

  // scales of this lane's key of a tile (int8)
  float ks = 0.f, vs = 1.f;
  auto scales = [&](int tile) {
    const int key = tile * TK + lane;
    ks = 0.f, vs = 1.f;
    if (key < ch.kv) {
      const int64_t r = pool_row(a.p, b, g, key);
      ks = __ldg(a.p.ks + r);
      vs = __ldg(a.p.vs + r);
    }
  };
  if (Q8 && t0 + warp < t1) scales(t0 + warp);

  // Q fragments: rows g8 and g8 + 8 of each row tile; k-step s
  uint32_t qa[MT][8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = 16 * mt + 8 * hf + g8, i = r / a.rep;
      const bool in = i < ch.n;
      const T* src = static_cast<const T*>(a.q) + ((ch.q0 + (in ? i : 0)) * a.hq + g * a.rep + r % a.rep) * D;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        if constexpr (Q8) {  // dims 32 qd + 4 s .. + 3
          const uint2 w = in ? __ldg(reinterpret_cast<const uint2*>(src + 32 * qd + 4 * s)) : make_uint2(0, 0);
          qa[mt][s][hf] = w.x;
          qa[mt][s][2 + hf] = w.y;
        } else {  // dims 16 s + 2 qd, + 1 and 8 further on
          qa[mt][s][hf] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * s + 2 * qd)) : 0u;
          qa[mt][s][2 + hf] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * s + 8 + 2 * qd)) : 0u;
        }
      }
    }

  float m[MT][2], l[MT][2], o[MT][16][4];
  int lim[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int i = (16 * mt + 8 * hf + g8) / a.rep;
      m[mt][hf] = -INFINITY;
      l[mt][hf] = 0.f;
      lim[mt][hf] = i < ch.n ? before + i + 1 : 0;
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.f;
  }

  const int mi = lane >> 3, ri = lane & 7;
  int st = 0;
  uint32_t ph = 0;
  for (int tile = t0 + warp; tile < t1; tile += WARPS) {
    if (!__all_sync(0xffffffffu, wait(bar + 8 * st, ph, err))) break;
    const uint32_t kt = ring + st * STAGE, vt = kt + TILE;
    const int k0 = tile * TK;
    float sc[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[mt][n][0] = sc[mt][n][1] = sc[mt][n][2] = sc[mt][n][3] = 0.f;
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int key = 8 * n + g8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 w = lds16(kt + key * 128 + (((2 * qd + h) ^ (key & 7)) << 4));
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t b0, b1;
            widen<T>(ww[x], b0, b1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma<T>(sc[mt][n], qa[mt][4 * h + x], b0, b1);
          }
        }
      }
    } else {
      if (k0 + TK > ch.kv) {  // value rows behind the cache's end must not meet a zero as a NaN
        for (int i = (ch.kv - k0) * 8 + lane; i < TK * 8; i += 32) {
          sts16(vt + i * 16, make_uint4(0, 0, 0, 0));
          sts16(vt + TILE / 2 + i * 16, make_uint4(0, 0, 0, 0));
        }
        __syncwarp();
      }
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const int row = (mi >> 1) * 8 + ri, cc = 2 * (s & 3) + (mi & 1);
        uint32_t w[4];
        ldsm(kt + (s >> 2) * (TILE / 2) + row * 128 + ((cc ^ (row & 7)) << 4), w);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma<T>(sc[mt][0], qa[mt][s], w[0], w[1]);
          mma<T>(sc[mt][1], qa[mt][s], w[2], w[3]);
        }
      }
    }
    // scores in log2 units; this lane holds keys 8 n + 2 qd, + 1 of rows g8 and g8 + 8
    float rv[NT][2];
    if constexpr (Q8) {
      const float kc = ks * a.c, lv = __log2f(vs), iv = 1.f / vs;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = __shfl_sync(0xffffffffu, kc, 8 * n + 2 * qd + e);
          const float v = __shfl_sync(0xffffffffu, lv, 8 * n + 2 * qd + e);
          rv[n][e] = __shfl_sync(0xffffffffu, iv, 8 * n + 2 * qd + e);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            sc[mt][n][e] = fmaf(sc[mt][n][e], f, v);
            sc[mt][n][2 + e] = fmaf(sc[mt][n][2 + e], f, v);
          }
        }
      if (tile + WARPS < t1) scales(tile + WARPS);
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][n][e] *= a.c;
    }
    const bool masked = k0 + TK > before + 1;
    uint32_t pa_[MT][NT / 2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = sc[mt][n][2 * hf + e];
            if (masked && k0 + 8 * n + 2 * qd + e >= lim[mt][hf]) x = -INFINITY;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[mt][hf], mx);
        const float f = m[mt][hf] == -INFINITY ? 0.f : ex2(m[mt][hf] - mn);
        m[mt][hf] = mn;
        const float sub = mn == -INFINITY ? 0.f : mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float x = ex2(sc[mt][n][2 * hf] - sub), y = ex2(sc[mt][n][2 * hf + 1] - sub);
          if constexpr (Q8) {
            // a key that the row does not see has no part in its sum, whatever its scale is
            sum += masked && x == 0.f ? 0.f : x * rv[n][0];
            sum += masked && y == 0.f ? 0.f : y * rv[n][1];
          } else {
            sum += x + y;
          }
          pa_[mt][n / 2][2 * (n & 1) + hf] = pack2<PT>(x, y);
        }
        l[mt][hf] = l[mt][hf] * f + sum;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          o[mt][n][2 * hf] *= f;
          o[mt][n][2 * hf + 1] *= f;
        }
      }
    }
    // O += P V
    if constexpr (Q8) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t w[4][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // keys 2 qd, 2 qd + 1, 2 qd + 8, 2 qd + 9
          const int key = 16 * kk + 2 * qd + (x & 1) + 8 * (x >> 1);
          const uint4 u = lds16(vt + key * 128 + ((g8 ^ (key & 7)) << 4));
          w[x][0] = u.x, w[x][1] = u.y, w[x][2] = u.z, w[x][3] = u.w;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)  // dims 16 g8 + 4 x .. + 3
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t b0a, b0b, b1a, b1b;
            widen<PT>(prmt(w[0][x], w[1][x], e ? 0x7362u : 0x5140u), b0a, b0b);
            widen<PT>(prmt(w[2][x], w[3][x], e ? 0x7362u : 0x5140u), b1a, b1b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma<PT>(o[mt][4 * x + 2 * e], pa_[mt][kk], b0a, b1a);
              mma<PT>(o[mt][4 * x + 2 * e + 1], pa_[mt][kk], b0b, b1b);
            }
          }
      }
    } else {
#pragma unroll
      for (int n = 0; n < 16; n += 2) {
        const int row = (mi & 1) * 8 + ri, cc = (n + (mi >> 1)) & 7;
        uint32_t w[4];
        ldsm_t(vt + (n >> 3) * (TILE / 2) + row * 128 + ((cc ^ (row & 7)) << 4), w);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma<PT>(o[mt][n], pa_[mt][0], w[0], w[1]);
          mma<PT>(o[mt][n + 1], pa_[mt][0], w[2], w[3]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0 && tile + STAGES * WARPS < t1) fetch(tile + STAGES * WARPS, st);
    if (++st == STAGES) st = 0, ph ^= 1;
  }

  // ---- the warps meet: O [row][dim] in the ring, which nobody fills any more
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float s = l[mt][hf];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (qd == 0) {
        sm_m[warp][16 * mt + 8 * hf + g8] = m[mt][hf];
        sm_l[warp][16 * mt + 8 * hf + g8] = s;
      }
    }
  __syncthreads();
  const int rows = min(ROWS, ch.n * a.rep);
  float* part = reinterpret_cast<float*>(smem);  // [WARPS][rows][D]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = 16 * mt + 8 * hf + g8;
      if (r >= rows) continue;
      float* dst = part + (warp * rows + r) * D;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const float x = o[mt][n][2 * hf], y = o[mt][n][2 * hf + 1];
        if constexpr (Q8) {  // column 2 qd + e of tile n is dim 16 (2 qd + e) + n
          dst[32 * qd + n] = x;
          dst[32 * qd + 16 + n] = y;
        } else {
          *reinterpret_cast<float2*>(dst + 8 * n + 2 * qd) = make_float2(x, y);
        }
      }
    }
  __syncthreads();
  // every row of this CTA in units of its maximum
  for (int x = threadIdx.x; x < rows * (D / 4); x += WARPS * 32) {
    const int r = x >> 5, d = (x & 31) * 4;
    float M = -INFINITY, Ls = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_m[w][r]);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (sm_m[w][r] == -INFINITY && !(sm_l[w][r] != 0.f)) continue;
      const float f = ex2(sm_m[w][r] - M);
      const float4 y = *reinterpret_cast<const float4*>(part + (w * rows + r) * D + d);
      Ls += sm_l[w][r] * f;
      v.x += y.x * f, v.y += y.y * f, v.z += y.z * f, v.w += y.w * f;
    }
    *reinterpret_cast<float4*>(part + r * D + d) = v;  // warp 0's place, read by this thread alone
    if (d == 0) cta_m[r] = M, cta_l[r] = Ls;
  }
  // ---- the CTAs meet: each finishes its share of the rows
  if (S > 1) cluster_sync();
  else __syncthreads();
  for (int r = rank * WARPS + warp; r < rows; r += S * WARPS) {
    const int i = r / a.rep;
    float M = -INFINITY, Ls = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (S == 1) {
      Ls = cta_l[r];
      v = *reinterpret_cast<const float4*>(part + r * D + 4 * lane);
    } else {
      // lane z holds part z's maximum and sum
      float mz = -INFINITY, lz = 0.f;
      if (lane < S) {
        mz = ld_cluster(mapa(smem_u32(&cta_m[r]), lane));
        lz = ld_cluster(mapa(smem_u32(&cta_l[r]), lane));
      }
      M = mz;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
      const float fz = mz == -INFINITY && !(lz != 0.f) ? 0.f : ex2(mz - M);
      const uint32_t at = smem_u32(part + r * D + 4 * lane);
#pragma unroll 8
      for (int z = 0; z < S; ++z) {
        const float f = __shfl_sync(0xffffffffu, fz, z), lp = __shfl_sync(0xffffffffu, lz, z);
        const float4 y = ld_cluster16(mapa(at, z));
        if (f != 0.f || lp != 0.f) {
          Ls += lp * f;
          v.x += y.x * f, v.y += y.y * f, v.z += y.z * f, v.w += y.w * f;
        }
      }
    }
    const float w[4] = {Ls == 0.f ? 0.f : v.x / Ls, Ls == 0.f ? 0.f : v.y / Ls, Ls == 0.f ? 0.f : v.z / Ls,
                        Ls == 0.f ? 0.f : v.w / Ls};
    bool fine = fabsf(Ls) < INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) fine = fine && fabsf(w[e]) < INFINITY;
    const int64_t at = ((ch.q0 + i) * a.hq + g * a.rep + r % a.rep) * D;
    // a value that is not finite may come from a row the token does not see (0 x NaN): such
    // rows are computed again, key by key
    if (__all_sync(0xffffffffu, fine))
      reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at)[lane] = make_uint2(pack2<T>(w[0], w[1]), pack2<T>(w[2], w[3]));
    else
      attend_row<T, Q8>(a.p, b, g, before + i + 1, static_cast<const T*>(a.q) + at, a.c, static_cast<T*>(a.out) + at);
  }
  if (S > 1) cluster_sync();  // nobody leaves while another reads its part
}

// Key splits (CTAs of a cluster) of `units` (sequence, kv head) pairs with up to
// `tiles` key tiles: the fewest rounds over the SMs' CTA places times the tiles a
// warp takes, plus what a CTA costs to start and to meet the others (about 12
// tiles of a warp).
int key_splits(int64_t units, int64_t tiles) {
  const int64_t places = 2 * (int64_t)sm_count();
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 8; s *= 2) {
    if (s > 1 && tiles < 2 * WARPS * s) break;
    const double rounds = (double)((units * s + places - 1) / places);
    const double c = rounds * ((double)tiles / (WARPS * s) + 12);
    if (c < cost - 1e-9) cost = c, best = s;
  }
  return best;
}

template <typename T, bool Q8, int MT>
dial_status launch(const void* q, const PagedView& p, void* out, int hq, int64_t max_kv, float c, cudaStream_t st) {
  constexpr auto kern = paged_attention_rows_kernel<T, Q8, MT>;
  constexpr int smem = RING + 1024;
  constexpr int TK = Q8 ? 32 : 16;
  const int64_t rows = (p.n_pages * p.hkv) << p.log2_page;
  CUtensorMap km, vm;
  const int box = std::min(1 << p.log2_page, TK);
  dial_status s = make_byte_map(&km, p.k, rows, Q8 ? 128 : 256, 128, box, 128);
  if (s == DIAL_OK) s = make_byte_map(&vm, p.v, rows, Q8 ? 128 : 256, 128, box, 128);
  if (s != DIAL_OK) return s;
  cudaError_t e = ensure_smem<kern>(smem);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attention_rows_kernel)");
  const int64_t units = (int64_t)p.n_seqs * p.hkv;
  const int S = key_splits(units, (max_kv + TK - 1) / TK);
  if (units * S >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many sequences and heads (%lld)", (long long)units);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * S));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const Args a{p, hq, hq / p.hkv, c, q, out};
  e = cudaLaunchKernelEx(&cfg, kern, km, vm, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, "paged_attention_rows_kernel");
  }
  return check_launch("paged_attention_rows_kernel");
}

template <typename T, bool Q8>
dial_status launch_mt(const void* q, const PagedView& p, void* out, int hq, int64_t max_kv, float c, cudaStream_t st) {
  return (int64_t)p.max_q * (hq / p.hkv) <= 16 ? launch<T, Q8, 1>(q, p, out, hq, max_kv, c, st)
                                               : launch<T, Q8, 2>(q, p, out, hq, max_kv, c, st);
}

}  // namespace

dial_status launch_paged_attention(const void* q, const PagedView& p, int format, void* out, dial_dtype dt,
                                   int hq, int64_t max_kv, float scale, cudaStream_t st) {
  const float c = (float)((double)scale * 1.4426950408889634);
  const bool q8 = format == DIAL_KV_INT8;
  if ((int64_t)p.max_q * (hq / p.hkv) > 32) return launch_paged_attention_tiles(q, p, format, out, dt, hq, max_kv, c, st);
  if (dt == DIAL_F16)
    return q8 ? launch_mt<__half, true>(q, p, out, hq, max_kv, c, st) : launch_mt<__half, false>(q, p, out, hq, max_kv, c, st);
  return q8 ? launch_mt<__nv_bfloat16, true>(q, p, out, hq, max_kv, c, st)
            : launch_mt<__nv_bfloat16, false>(q, p, out, hq, max_kv, c, st);
}

}  // namespace dial
