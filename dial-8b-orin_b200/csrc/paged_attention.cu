// Attention over a paged KV cache for few query rows (decoding, drafted tokens):
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t.k_j - m_t),  c = scale log2(e),
//
// over the cache rows j up to the token's own.  The rows of a sequence and kv head
// (token x query head of the group, at most 32) share every key, so the work is
// bound by the bytes of the cache.
//
// A CTA takes a share of the key tiles of one (sequence, kv head); its four warps
// take tiles in turn, each through a ring of its own of 8 KB stages that one lane
// fills by TMA (SWIZZLE_128B, boxes inside a page).  mma.sync m16n8k16 does the
// products, with the query rows on its N side, eight to a tile, so that few rows
// waste little:
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 dims x 8 rows] += V^T P^T;
// S^T's 8 x 8 blocks become P^T's operand by movmatrix.  A row's maximum in use
// moves only when a score passes it by 2^8 (a vote; the exchange over the lanes is
// rare); P's range is in paged_attention.cuh.
//   16-bit pages: 16 keys a tile, operands by ldmatrix (V transposed).
//   int8 pages: 32 keys a tile, widened to f16 in registers.  The order of the 128
//   dims in K Q^T is free as long as Q follows it: a lane takes 16 consecutive bytes
//   of a key, so two 16-byte loads a key feed 8 k-steps; V's 4 x 4 byte blocks are
//   transposed with byte permutes, and the dims of O come out permuted.  bf16 queries
//   become f16 times one power of two for all rows, chosen by their largest value: 34
//   bits below it are kept.  Scales as in paged_attention_tiles.cu: k_s on the score,
//   log2 v_s in the exponent, 1 / v_s in the row sum.
// The warps' (m, l, O) meet in shared memory, the CTAs' in the cluster's: no
// workspace, no counters, and the same result whatever the timing.
// 32 sequences of 2049 int8 rows (8 kv heads, one token each) take 33 us (139 MB, 4.2 TB/s,
// 20 us of it streaming); 16 with 5 tokens over up to 8200 bf16 rows 48 us (233 MB, 4.9
// TB/s); one sequence of 2049 f16 rows 7.6 us, the chain length, page, tile, meeting.
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
// A CTA's warps, their rings and how many CTAs share an SM (about 192 KB in flight on it).
template <bool Q8, int NR>
struct Cfg {
  static constexpr int WARPS = Q8 && NR == 1 ? 8 : 4;
  static constexpr int TK = Q8 && NR > 1 ? 32 : 16;  // keys per tile
  static constexpr int TILE = TK * (Q8 ? 128 : 256); // bytes of a K or V tile
  static constexpr int STAGE = 2 * TILE;
  static constexpr int STAGES = !Q8 && NR == 1 ? 2 : 3;
  static constexpr int PER_SM = !Q8 && NR == 1 ? 3 : 2;
  static constexpr int RING = WARPS * STAGES * STAGE;
};

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

// an 8 x 8 matrix of 16-bit values, transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// NR: 8-row tiles of query rows (rows of the chunk = token * rep + head)
template <typename T, bool Q8, int NR>
__global__ void __launch_bounds__((Cfg<Q8, NR>::WARPS * 32), (Cfg<Q8, NR>::PER_SM))
    paged_attention_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                const Args a) {
  using L = Cfg<Q8, NR>;
  constexpr int TK = L::TK, WARPS = L::WARPS, TILE = L::TILE, STAGE = L::STAGE, STAGES = L::STAGES;
  constexpr int KT = TK / 16;       // 16-key tiles of the scores
  constexpr int ROWS = 8 * NR;
  using MT = typename std::conditional<Q8, __half, T>::type;  // operands
  constexpr float LIFT = kLift<MT>;
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
  const int mine = t0 + warp;                          // this warp's tiles: mine + i WARPS
  const int box = min(1 << a.p.log2_page, TK);

  // Q: row 8 n + g8; k-step s (asked for before the tiles, which would keep it waiting)
  uint32_t qb[NR][8][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = 8 * n + g8, i = r / a.rep;
    const bool in = i < ch.n;
    const T* src = static_cast<const T*>(a.q) + ((ch.q0 + (in ? i : 0)) * a.hq + g * a.rep + r % a.rep) * D;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if constexpr (Q8) {  // dims 32 qd + 4 s .. + 3
        const uint2 w = in ? __ldg(reinterpret_cast<const uint2*>(src + 32 * qd + 4 * s)) : make_uint2(0, 0);
        qb[n][s][0] = w.x;
        qb[n][s][1] = w.y;
      } else {  // dims 16 s + 2 qd, + 1 and 8 further on
        qb[n][s][0] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * s + 2 * qd)) : 0u;
        qb[n][s][1] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * s + 8 + 2 * qd)) : 0u;
      }
    }
  }

  // pool rows of this warp's tiles, 32 tiles at a time, a lane each (two for an int8 tile
  // over two 16-row pages): for the copies, and for the scales, which are behind them
  int row0 = 0, row1 = 0, srow0 = 0, srow1 = 0;
  auto look_up = [&](int i, int& r0, int& r1) {  // tiles i .. i + 31 of this warp
    const int k = (mine + (i + lane) * WARPS) * TK;
    if (mine + (i + lane) * WARPS < t1) {
      r0 = (int)pool_row(a.p, b, g, k);
      if (Q8 && box < TK && k + box < ch.kv) r1 = (int)pool_row(a.p, b, g, k + box);
    }
  };
  auto fetch = [&](int i, int st) {  // tile i of this warp (the whole warp calls)
    const int r0 = __shfl_sync(0xffffffffu, row0, i & 31), r1 = __shfl_sync(0xffffffffu, row1, i & 31);
    if (lane == 0) {
      const uint32_t dst = ring + st * STAGE, fb = bar + 8 * st;
      if constexpr (Q8) {
        const bool both = box < TK && (mine + i * WARPS) * TK + box < ch.kv;
        mbar_expect_tx(fb, (uint32_t)(2 * (both ? TK : box) * 128));
        load_2d(dst, &kmap, fb, 0, r0);
        load_2d(dst + TILE, &vmap, fb, 0, r0);
        if (both) {
          load_2d(dst + box * 128, &kmap, fb, 0, r1);
          load_2d(dst + TILE + box * 128, &vmap, fb, 0, r1);
        }
      } else {
        mbar_expect_tx(fb, STAGE);
        load_3d(dst, &kmap, fb, 0, r0, 0);
        load_3d(dst + TILE, &vmap, fb, 0, r0, 0);
      }
    }
    __syncwarp();
  };
  const int count = mine < t1 ? (t1 - mine + WARPS - 1) / WARPS : 0;
  look_up(0, row0, row1);
  srow0 = row0, srow1 = row1;
  for (int s = 0; s < STAGES; ++s)
    if (s < count) fetch(s, s);

  // scales of this lane's keys of tile i (int8): g8 + 8 x.  Rows behind the cache's end are
  // in the same page, and masked.
  float ks[2 * KT], vs[2 * KT];
  auto scales = [&](int i) {
    if ((i & 31) == 0 && i) look_up(i, srow0, srow1);
    const int r0 = __shfl_sync(0xffffffffu, srow0, i & 31), r1 = __shfl_sync(0xffffffffu, srow1, i & 31);
    const bool both = box == TK || (mine + i * WARPS) * TK + box < ch.kv;
#pragma unroll
    for (int x = 0; x < 2 * KT; ++x) {
      const int r = x < KT || box == TK ? r0 + 8 * x + g8 : r1 + 8 * (x - KT) + g8;
      const bool in = x < KT || both;
      ks[x] = in ? __ldg(a.p.ks + r) : 0.f;
      vs[x] = in ? __ldg(a.p.vs + r) : 1.f;
    }
  };
  if (Q8 && count) scales(0);

  float c = a.c;
  if constexpr (Q8 && std::is_same<T, __nv_bfloat16>::value) {  // to f16, the largest to 2^10 .. 2^11
    float top = 0.f;
    auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
    auto hi = [](uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); };
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = fabsf(lo(qb[n][s][e])), y = fabsf(hi(qb[n][s][e]));
          if (x < INFINITY) top = fmaxf(top, x);
          if (y < INFINITY) top = fmaxf(top, y);
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = max((int)(__float_as_uint(top) >> 23) - 127 - 10, -100);  // up to 117
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    c *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) qb[n][s][x] = pack2<__half>(lo(qb[n][s][x]) * down, hi(qb[n][s][x]) * down);
  }

  float m[NR][2], l[NR][2], o[NR][8][4];  // rows 8 n + 2 qd, + 1
  int lim[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = (8 * n + 2 * qd + e) / a.rep;
      m[n][e] = -INFINITY;
      l[n][e] = 0.f;
      lim[n][e] = i < ch.n ? before + i + 1 : 0;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) o[n][x][0] = o[n][x][1] = o[n][x][2] = o[n][x][3] = 0.f;
  }

  const int mi = lane >> 3, ri = lane & 7;
  int st = 0;
  uint32_t ph = 0;
  for (int i = 0; i < count; ++i) {
    const int tile = mine + i * WARPS, k0 = tile * TK;
    if (!__all_sync(0xffffffffu, wait(bar + 8 * st, ph, err))) break;
    const uint32_t kt = ring + st * STAGE, vt = kt + TILE;
    float sc[NR][KT][4];  // keys 16 x + g8 (0, 1) and + 8 (2, 3), rows 2 qd, + 1
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int x = 0; x < KT; ++x) sc[n][x][0] = sc[n][x][1] = sc[n][x][2] = sc[n][x][3] = 0.f;
    if constexpr (Q8) {
#pragma unroll
      for (int x = 0; x < KT; ++x) {
        const int key = 16 * x + g8;  // and key + 8: the same place in its group of eight
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t at = kt + key * 128 + (((2 * qd + h) ^ (key & 7)) << 4);
          const uint4 u = lds16(at), w = lds16(at + 1024);
          const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t f[4];
            widen<__half>(uu[y], f[0], f[2]);
            widen<__half>(ww[y], f[1], f[3]);
#pragma unroll
            for (int n = 0; n < NR; ++n) mma<MT>(sc[n][x], f, qb[n][4 * h + y][0], qb[n][4 * h + y][1]);
          }
        }
      }
    } else {
      if (k0 + TK > ch.kv) {  // value rows behind the cache's end must not meet a zero as a NaN
        for (int x = (ch.kv - k0) * 8 + lane; x < TK * 8; x += 32) {
          sts16(vt + x * 16, make_uint4(0, 0, 0, 0));
          sts16(vt + TILE / 2 + x * 16, make_uint4(0, 0, 0, 0));
        }
        __syncwarp();
      }
#pragma unroll
      for (int s = 0; s < 8; ++s) {  // keys ri and ri + 8, chunks 2 s and 2 s + 1
        const int row = (mi & 1) * 8 + ri, cc = 2 * (s & 3) + (mi >> 1);
        uint32_t f[4];
        ldsm(kt + (s >> 2) * (TILE / 2) + row * 128 + ((cc ^ (row & 7)) << 4), f);
#pragma unroll
        for (int n = 0; n < NR; ++n) mma<MT>(sc[n][0], f, qb[n][s][0], qb[n][s][1]);
      }
    }
    // scores in log2 units (16-bit pages: before the factor c), those that a row does not see
    // at minus infinity
    const bool masked = k0 + TK > before + 1;
    float rv[2 * KT];
    if constexpr (Q8) {
#pragma unroll
      for (int x = 0; x < 2 * KT; ++x) {
        const float kc = ks[x] * c, lv = lg2(vs[x]);
        rv[x] = rcp(vs[x]);
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) sc[n][x / 2][2 * (x & 1) + e] = fmaf(sc[n][x / 2][2 * (x & 1) + e], kc, lv);
      }
      if (i + 1 < count) scales(i + 1);
    }
    if (masked) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int x = 0; x < KT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + 16 * x + 8 * (e >> 1) + g8 >= lim[n][e & 1]) sc[n][x][e] = -INFINITY;
    }
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(sc[n][0][e], sc[n][0][2 + e]);
#pragma unroll
        for (int x = 1; x < KT; ++x) mx = fmaxf(mx, fmaxf(sc[n][x][e], sc[n][x][2 + e]));
        grow |= (Q8 ? mx : mx * c) > m[n][e] + (kGrow + LIFT);
      }
    if (__any_sync(0xffffffffu, grow)) {  // rare: the rows' maxima move
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int x = 0; x < KT; ++x) mx = fmaxf(mx, fmaxf(sc[n][x][e], sc[n][x][2 + e]));
#pragma unroll
          for (int z = 4; z < 32; z <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, z));
          const float mn = fmaxf(m[n][e], (Q8 ? mx : mx * c) - LIFT);
          const float f = m[n][e] == -INFINITY ? 0.f : ex2(m[n][e] - mn);
          m[n][e] = mn;
          l[n][e] *= f;
#pragma unroll
          for (int x = 0; x < 8; ++x) o[n][x][e] *= f, o[n][x][2 + e] *= f;
        }
    }
    uint32_t pb[NR][KT][2];  // P^T: keys 2 qd, + 1 (and 8 further on), row g8
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float s0 = m[n][0] == -INFINITY ? 0.f : m[n][0], s1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
      for (int x = 0; x < KT; ++x) {
        float* v = sc[n][x];
        if constexpr (Q8)
          v[0] = ex2(v[0] - s0), v[1] = ex2(v[1] - s1), v[2] = ex2(v[2] - s0), v[3] = ex2(v[3] - s1);
        else
          v[0] = ex2(fmaf(v[0], c, -s0)), v[1] = ex2(fmaf(v[1], c, -s1)), v[2] = ex2(fmaf(v[2], c, -s0)), v[3] = ex2(fmaf(v[3], c, -s1));
        if constexpr (Q8) {
          if (masked) {  // a key that the row does not see has no part in its sum, whatever its scale is
            l[n][0] += (v[0] == 0.f ? 0.f : v[0] * rv[2 * x]) + (v[2] == 0.f ? 0.f : v[2] * rv[2 * x + 1]);
            l[n][1] += (v[1] == 0.f ? 0.f : v[1] * rv[2 * x]) + (v[3] == 0.f ? 0.f : v[3] * rv[2 * x + 1]);
          } else {
            l[n][0] = fmaf(v[0], rv[2 * x], fmaf(v[2], rv[2 * x + 1], l[n][0]));
            l[n][1] = fmaf(v[1], rv[2 * x], fmaf(v[3], rv[2 * x + 1], l[n][1]));
          }
        } else {
          l[n][0] += v[0] + v[2];
          l[n][1] += v[1] + v[3];
        }
        // (rounded to the operands' type: a second part for the rest, as dial_attention has, would
        // double the products; against 64 bits the error is 5 % above that of f32 probabilities)
        pb[n][x][0] = transpose8(pack2<MT>(v[0], v[1]));
        pb[n][x][1] = transpose8(pack2<MT>(v[2], v[3]));
      }
    }
    // O^T += V^T P^T
    if constexpr (Q8) {
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        uint32_t w[4][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // keys 2 qd, 2 qd + 1, 2 qd + 8, 2 qd + 9
          const int key = 16 * kk + 2 * qd + (x & 1) + 8 * (x >> 1);
          const uint4 u = lds16(vt + key * 128 + ((g8 ^ (key & 7)) << 4));
          w[x][0] = u.x, w[x][1] = u.y, w[x][2] = u.z, w[x][3] = u.w;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)  // dims 16 g8 + 4 x .. + 3, two to a 16-dim tile
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t f[4];
            widen<__half>(prmt(w[0][x], w[1][x], e ? 0x7362u : 0x5140u), f[0], f[1]);
            widen<__half>(prmt(w[2][x], w[3][x], e ? 0x7362u : 0x5140u), f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NR; ++n) mma<MT>(o[n][2 * x + e], f, pb[n][kk][0], pb[n][kk][1]);
          }
      }
    } else {
#pragma unroll
      for (int x = 0; x < 8; ++x) {  // dims 16 x .. + 15: chunks 2 x (mi & 1), keys ri + 8 (mi >> 1)
        const int row = (mi >> 1) * 8 + ri, cc = (2 * x + (mi & 1)) & 7;
        uint32_t f[4];
        ldsm_t(vt + (x >> 2) * (TILE / 2) + row * 128 + ((cc ^ (row & 7)) << 4), f);
#pragma unroll
        for (int n = 0; n < NR; ++n) mma<MT>(o[n][x], f, pb[n][0][0], pb[n][0][1]);
      }
    }
    __syncwarp();  // every lane has read the stage
    const int next = i + STAGES;
    if (next < count) {
      if ((next & 31) == 0) look_up(next, row0, row1);
      fetch(next, st);
    }
    if (++st == STAGES) st = 0, ph ^= 1;
  }

  // ---- the warps meet: O [row][dim] in the ring, which nobody fills any more
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[n][e];
#pragma unroll
      for (int z = 4; z < 32; z <<= 1) s += __shfl_xor_sync(0xffffffffu, s, z);
      if (g8 == 0) {
        sm_m[warp][8 * n + 2 * qd + e] = m[n][e];
        sm_l[warp][8 * n + 2 * qd + e] = s;
      }
    }
  __syncthreads();
  const int rows = min(ROWS, ch.n * a.rep);
  float* part = reinterpret_cast<float*>(smem);  // [WARPS][rows][D]
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * n + 2 * qd + e;
      if (r >= rows) continue;
      float* dst = part + (warp * rows + r) * D;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if constexpr (Q8) {  // dims 16 g8 + 2 x, + 1
          *reinterpret_cast<float2*>(dst + 16 * g8 + 2 * x) = make_float2(o[n][x][e], o[n][x][2 + e]);
        } else {             // dims 16 x + g8, + 8
          dst[16 * x + g8] = o[n][x][e];
          dst[16 * x + g8 + 8] = o[n][x][2 + e];
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
      M = cta_m[r];
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
    bool fine = fabsf(Ls) < INFINITY && (Q8 || in_range<MT>(Ls, M));
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

// Key splits (CTAs of a cluster) of `units` (sequence, kv head) pairs with up to `tiles`
// key tiles: the least of rounds over the SMs' CTA places times (tiles a warp takes + 5),
// as a CTA's start and its meeting with the others cost about five tiles.  Rounds count
// in fractions, as lengths differ and places fill as they come free: 16 ragged sequences
// of up to 8200 rows took 96 / 61 / 49 / 56 us with 1 / 2 / 4 / 8 CTAs each, 32 of 2049
// rows (int8) 33 / 42 / 56 / 83.
int key_splits(int64_t units, int64_t tiles, int per_sm, int warps) {
  const double places = (double)per_sm * sm_count();
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 8; s *= 2) {
    if (s > 1 && tiles < 2 * warps * s) break;
    const double c = std::max(1.0, units * s / places) * ((double)tiles / (warps * s) + 5);
    if (c < cost - 1e-9) cost = c, best = s;
  }
  return best;
}

template <typename T, bool Q8, int NR>
dial_status launch(const void* q, const PagedView& p, void* out, int hq, int64_t max_kv, float c, cudaStream_t st) {
  constexpr auto kern = paged_attention_rows_kernel<T, Q8, NR>;
  using L = Cfg<Q8, NR>;
  constexpr int smem = L::RING + 1024, TK = L::TK;
  const int64_t rows = (p.n_pages * p.hkv) << p.log2_page;
  CUtensorMap km, vm;
  const int box = std::min(1 << p.log2_page, TK);
  dial_status s = Q8 ? make_byte_map(&km, p.k, rows, 128, 128, box, 128) : make_halves_map(&km, p.k, rows, box);
  if (s == DIAL_OK) s = Q8 ? make_byte_map(&vm, p.v, rows, 128, 128, box, 128) : make_halves_map(&vm, p.v, rows, box);
  if (s != DIAL_OK) return s;
  cudaError_t e = ensure_smem<kern>(smem);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attention_rows_kernel)");
  const int64_t units = (int64_t)p.n_seqs * p.hkv;
  const int S = key_splits(units, (max_kv + TK - 1) / TK, L::PER_SM, L::WARPS);
  if (units * S >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many sequences and heads (%lld)", (long long)units);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * S));
  cfg.blockDim = dim3(L::WARPS * 32);
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
dial_status launch_rows(const void* q, const PagedView& p, void* out, int hq, int64_t max_kv, float c, cudaStream_t st) {
  const int64_t rows = (int64_t)p.max_q * (hq / p.hkv);
  return rows <= 8    ? launch<T, Q8, 1>(q, p, out, hq, max_kv, c, st)
         : rows <= 16 ? launch<T, Q8, 2>(q, p, out, hq, max_kv, c, st)
         : rows <= 24 ? launch<T, Q8, 3>(q, p, out, hq, max_kv, c, st)
                      : launch<T, Q8, 4>(q, p, out, hq, max_kv, c, st);
}

}  // namespace

dial_status launch_paged_attention(const void* q, const PagedView& p, int format, void* out, dial_dtype dt,
                                   int hq, int64_t max_kv, float scale, cudaStream_t st) {
  const float c = (float)((double)scale * 1.4426950408889634);
  const bool q8 = format == DIAL_KV_INT8;
  if ((int64_t)p.max_q * (hq / p.hkv) > 32) return launch_paged_attention_tiles(q, p, format, out, dt, hq, max_kv, c, st);
  if (dt == DIAL_F16)
    return q8 ? launch_rows<__half, true>(q, p, out, hq, max_kv, c, st) : launch_rows<__half, false>(q, p, out, hq, max_kv, c, st);
  return q8 ? launch_rows<__nv_bfloat16, true>(q, p, out, hq, max_kv, c, st)
            : launch_rows<__nv_bfloat16, false>(q, p, out, hq, max_kv, c, st);
}

}  // namespace dial
