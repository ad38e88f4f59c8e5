// Attention of long chunks over a paged KV cache on the tcgen05 tensor cores.
//
// A CTA owns one kv head of one sequence and up to 256 query rows of it, in two
// tiles of 128: a row is (token, query head of the group), 128 / rep tokens a
// tile.  Keys go by in tiles of 128:
//   S = Q K^T   tcgen05.mma, both operands in shared memory, f32 in TMEM
//   P = 2^(c S - m)   one thread a row: its 128 scores come to registers, the row
//               maximum needs no exchange, P goes back over S as 16-bit pairs
//   O += P V    A = P from TMEM, B = V as the pages hold it ([key][dim], the
//               MN-major descriptor), f32 in TMEM
// While a warpgroup turns S into P for one tile, the tensor cores work on the
// other.  O is rescaled only when a row's maximum grew by more than 2^8 over the
// one in use (P's range is in paged_attention.cuh), by the
// thread that owns the row: S of a key tile is complete only after O += P V of
// the tile before, so nothing else touches O then.
//
// int8 pages: a warpgroup widens the codes to 16 bits (exact).  The key's scale
// multiplies its score column; the value's scale v goes into the exponent, P' =
// 2^(c k_s S + log2 v - m'), so that P' stays in [0, 2^15] whatever the scales
// are, and the row sum takes P' / v.
//
// TMEM (512 columns): S of the two tiles in [0, 256), O in [256, 512).
// Shared memory: Q (64 KB), a ring of 32 KB slots for K_0 V_0 K_1 V_1 .. and,
// for int8, a ring of 16 KB raw ones, rows of 128 bytes, SWIZZLE_128B.
// Few rows and many keys: the key tiles are split over a cluster of CTAs, whose
// (m, l, O) meet in distributed shared memory, so that no workspace is needed
// and the result does not depend on timing.
// 2048 tokens of 32 heads behind 14336 others in bf16 take 422 us, 1.22 PFLOP/s, at 1965 MHz
// (490, 1.05, once the power limit has lowered the clock); inside a CTA a key tile of 2 x 128
// rows takes 1.7 us, in which the tensor cores and the exponentials are busy alike (65 %), and
// 256 CTAs are 1.73 rounds over the SMs.  8 ragged int8 chunks of up to 777 tokens take 99.5
// us, 0.61 PFLOP/s (99 to 114 from run to run): widening the codes shares the shared memory's
// bandwidth with the MMAs' operands.
// Every mbarrier wait is bounded (1 s), flags DIAL_ERR_TIMEOUT and gives up.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "paged_attention.cuh"
#include "tma.cuh"

namespace dial {

namespace {

using namespace pa;
using namespace tma;

constexpr int KT = 128;             // keys per tile
constexpr int QT = 128;             // rows per query tile
constexpr int HALF = KT * 128;      // bytes of 128 rows x 64 dims of 16 bits
constexpr int SLOT = 2 * HALF;      // one K or V tile
constexpr int RAW = KT * 128;       // one int8 K or V tile

template <bool Q8>
struct Cfg {
  static constexpr int THREADS = Q8 ? 512 : 384;
  static constexpr int SLOTS = Q8 ? 3 : 4;
  static constexpr int RAWS = Q8 ? 3 : 0;
  static constexpr int Q_BYTES = 2 * SLOT;
  static constexpr int RING = Q_BYTES;
  static constexpr int RAW_OFF = RING + SLOTS * SLOT;
  static constexpr int SC_OFF = RAW_OFF + RAWS * RAW;  // [3][3][KT] f32: c k_s, log2 v_s, 1 / v_s
  static constexpr int ML_OFF = SC_OFF + (Q8 ? 3 * 3 * KT * 4 : 0);  // m, l of 256 rows
  static constexpr int BAR_OFF = ML_OFF + 2 * 2 * QT * 4;
  static constexpr int BYTES = BAR_OFF + 256 + 1024;
  static_assert(BYTES <= 227 * 1024, "shared memory budget");
  // registers: the softmax warpgroups' share after setmaxnreg; the sum equals the launch's
  static constexpr int REGS = Q8 ? 128 : 168, SOFT_REGS = Q8 ? 184 : 216, REST_REGS = 72;
  static_assert(REGS * (THREADS / 128) == 2 * SOFT_REGS + (THREADS / 128 - 2) * REST_REGS, "register split");
};

struct Args {
  PagedView p;
  int hq, rep, tpt;  // tokens per 128-row tile
  float c;           // scale log2(e)
  const void* q;
  void* out;
};

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Descriptors of SWIZZLE_128B tiles whose rows are 128 bytes (8-row atoms of 1024):
// K-major (Q, K: the row's 64 values run along K) and MN-major (V: they run along N;
// 8-key groups 1024 bytes apart, the two 64-dim blocks HALF apart).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// M = 128, N = 128, f32 accumulators; f16 (0) or bf16 (1) operands, B K-major or MN-major
__device__ constexpr uint32_t idesc(bool bf16, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 columns of the warp's 32 lanes (no wait)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// (a0 b0 + c0, a1 b1 + c1) in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// The t-th query tile (of two times 128 rows) of the batch: sequence by sequence, a chunk's
// last tile, which sees the most keys, first.  False behind the last.  By a whole warp, a
// sequence per lane.
__device__ __forceinline__ bool tile_of(const Args& a, int t, int& qt, int& b) {
  const int lane = threadIdx.x & 31, rows = 2 * a.tpt;
  const bool report = blockIdx.x == 0 && threadIdx.x < 32;
  bool found = false;
  for (int i = 0; i < a.p.n_seqs && (!found || report); i += 32) {
    int n = 0;
    if (i + lane < a.p.n_seqs) n = (chunk_of(a.p, i + lane, report).n + rows - 1) / rows;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sum > t);
    if (past && !found) {
      const int l = __ffs(past) - 1;
      b = i + l;
      qt = __shfl_sync(0xffffffffu, sum, l) - 1 - t;
      found = true;
    }
    t -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return found;
}

template <typename T, bool Q8>
__global__ void __launch_bounds__(Cfg<Q8>::THREADS, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap, const Args a) {
  using L = Cfg<Q8>;
  using PT = typename std::conditional<Q8, __half, T>::type;  // operands of P V
  constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value, kPBf = std::is_same<PT, __nv_bfloat16>::value;
  constexpr int NS = L::SLOTS;
  constexpr float LIFT = kLift<PT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_u32(smem), bars = base + L::BAR_OFF;
  float* sm_ml = reinterpret_cast<float*>(smem + L::ML_OFF);
  const uint32_t q_full = bars, o_full = bars + 8, v_fix = bars + 16, s_full = bars + 24, p_full = bars + 40;
  const uint32_t full = bars + 72, empty = full + 8 * NS, raw_full = empty + 8 * NS, raw_empty = raw_full + 8 * 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::BAR_OFF + 248);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* err = a.p.err;

  pdl_trigger();
  pdl_wait();

  // ---- this CTA's rows and keys
  const int S = (int)cluster_size(), rank = (int)cluster_rank();
  const int unit = blockIdx.x / S, g = unit % a.p.hkv;
  int qt, b;                                           // tile of its chunk, sequence
  if (!tile_of(a, unit / a.p.hkv, qt, b)) return;      // the grid is an upper bound
  const Chunk ch = chunk_of(a.p, b, false);
  const int i0 = qt * 2 * a.tpt;                       // first token (of the chunk) of this CTA
  const int ntok = min(ch.n - i0, 2 * a.tpt);          // its tokens
  const bool two = ntok > a.tpt;
  const int before = ch.kv - ch.n;                     // token i sees keys 0 .. before + i
  const int len = max(0, before + i0 + ntok);
  const int nkt = (len + KT - 1) / KT;
  const int j0 = (int)((int64_t)nkt * rank / S), nj = (int)((int64_t)nkt * (rank + 1) / S) - j0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(o_full, 1);
    mbar_init(v_fix, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + 8 * t, 1);
      mbar_init(p_full + 16 * t, 4);      // keys 0 .. 63
      mbar_init(p_full + 16 * t + 8, 4);  // keys 64 .. 127
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(full + 8 * s, Q8 ? 4 : 1);
      mbar_init(empty + 8 * s, 1);
    }
    if (Q8)
      for (int s = 0; s < 3; ++s) {
        mbar_init(raw_full + 8 * s, 1);
        mbar_init(raw_empty + 8 * s, 4);
      }
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REST_REGS));
    if (warp == 8) {
      // ------------------------------------------------ MMA issuer
      // The whole warp walks the loop and one lane issues: what is the same for all lanes stays in
      // uniform registers, where the MMA wants its descriptors, and an MMA costs few instructions.
      if (nj > 0) {
        const bool lead = elect();
        bool ok = wait(q_full, 0, err);
        const uint64_t qd = desc(base, 16), kd = desc(base + L::RING, 16), vd = desc(base + L::RING, HALF);
        auto step = [](int s) { return (uint64_t)((s >> 2) * (HALF >> 4) + 2 * (s & 3)); };  // 16 dims on
        auto score = [&](int slot, int t) {  // S_t = Q_t K^T
          const uint64_t q = qd + (uint64_t)(t * (SLOT >> 4)), k = kd + (uint64_t)(slot * (SLOT >> 4));
          if (lead) {
#pragma unroll
            for (int s = 0; s < 8; ++s) mma_ss(tmem + t * 128, q + step(s), k + step(s), idesc(kBf, false), s != 0);
            commit(s_full + 8 * t);
          }
          __syncwarp();
        };
        auto full_wait = [&](int u) { return wait(full + 8 * (u % NS), (uint32_t)(u / NS) & 1u, err); };
        ok = ok && full_wait(0);
        fence_after();
        if (ok) {
          score(0, 0);
          if (two) score(0, 1);
          if (lead) commit(empty);
          __syncwarp();
        }
        const int ntile = two ? 2 : 1;
        for (int j = 0; j < nj && ok; ++j) {
          const int v = 2 * j + 1, vslot = v % NS, kslot = (v + 1) % NS;
          const uint64_t vb = vd + (uint64_t)(vslot * (SLOT >> 4));
          for (int t = 0; t < ntile && ok; ++t) {
            if (t == 0) {
              ok = full_wait(v);
              if (!Q8 && (j0 + j + 1) * KT > ch.kv) ok = ok && wait(v_fix, 0, err);  // rows behind the cache's end
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ok = ok && wait(p_full + 16 * t + 8 * h, (uint32_t)j & 1u, err);
              fence_after();
              if (ok && lead) {
#pragma unroll
                for (int s = 4 * h; s < 4 * h + 4; ++s)
                  mma_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * s, vb + (uint64_t)(128 * s), idesc(kPBf, true), (j | s) != 0);
              }
              __syncwarp();
            }
            if (ok && j + 1 < nj) {
              if (t == 0) {
                ok = full_wait(v + 1);
                fence_after();
              }
              if (ok) score(kslot, t);
            }
          }
          if (ok && lead) {
            commit(empty + 8 * vslot);
            if (j + 1 < nj) commit(empty + 8 * kslot);
          }
          __syncwarp();
        }
        if (lead) commit(o_full);
        __syncwarp();
      }
    } else if (warp == 9) {
      // ------------------------------------------------ TMA producer
      if (nj > 0) {
        const int page = 1 << a.p.log2_page, box = min(page, KT), nbox = KT / box;
        if (lane == 0) {
          prefetch_map(&qmap);
          prefetch_map(&kmap);
          prefetch_map(&vmap);
          const uint32_t bytes = (uint32_t)(a.tpt * a.rep * 128);
          mbar_expect_tx(q_full, bytes * (two ? 4 : 2));
          for (int t = 0; t < (two ? 2 : 1); ++t)
            for (int h = 0; h < 2; ++h)
              load_3d(base + t * SLOT + h * HALF, &qmap, q_full, 128 * h, g * a.rep, (int)ch.q0 + i0 + t * a.tpt);
        }
        // a lane per box: (box of the tile, half of the 256-byte row); int8 rows have one half
        const int hb = Q8 ? 0 : lane & 1, bx = Q8 ? lane : lane >> 1;
        constexpr int R = Q8 ? L::RAWS : NS;
        for (int u = 0; u < 2 * nj; ++u) {
          const int key0 = (j0 + u / 2) * KT;
          const int n = min(nbox, (min(ch.kv - key0, KT) + box - 1) / box);  // boxes with rows of the sequence
          int row = 0;
          if (bx < n) {
            const int k = key0 + bx * box;
            row = (int)(((page_of(a.p, b, k >> a.p.log2_page) * a.p.hkv + g) << a.p.log2_page) + (k & (page - 1)));
          }
          const uint32_t fb = (Q8 ? raw_full : full) + 8 * (u % R), eb = (Q8 ? raw_empty : empty) + 8 * (u % R);
          if (!__all_sync(0xffffffffu, wait(eb, ((uint32_t)(u / R) & 1u) ^ 1u, err))) break;
          if (lane == 0) mbar_expect_tx(fb, (uint32_t)(n * box * (Q8 ? 128 : 256)));
          __syncwarp();
          if (bx < n) {
            const uint32_t dst = Q8 ? base + L::RAW_OFF + (u % R) * RAW + bx * box * 128
                                    : base + L::RING + (u % R) * SLOT + hb * HALF + bx * box * 128;
            load_2d(dst, (u & 1) ? &vmap : &kmap, fb, 128 * hb, row);
          }
          __syncwarp();
        }
        // value rows behind the cache's end must not meet a zero probability as a NaN: they
        // become zeros (int8 codes are finite whatever they are)
        const int u = 2 * nj - 1, end = ch.kv - (j0 + nj - 1) * KT;
        if (!Q8 && end < KT && __all_sync(0xffffffffu, wait(full + 8 * (u % NS), (uint32_t)(u / NS) & 1u, err))) {
          const uint32_t slot = base + L::RING + (uint32_t)(u % NS) * SLOT;
          for (int i = end * 8 + lane; i < KT * 8; i += 32) {
            sts16(slot + i * 16, make_uint4(0, 0, 0, 0));
            sts16(slot + HALF + i * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) arrive(v_fix);
        }
      }
    } else if (Q8 && warp >= 12) {
      // ------------------------------------------------ int8 -> 16 bits: a thread per key row
      const int row = threadIdx.x - 384, sw = row & 7;
      float ks = 0.f, vs = 0.f;
      auto scales = [&](int j) {  // of key row `row` of tile j
        const int key = (j0 + j) * KT + row;
        ks = vs = 0.f;
        if (key < ch.kv) {
          const int64_t r = pool_row(a.p, b, g, key);
          ks = __ldg(a.p.ks + r);
          vs = __ldg(a.p.vs + r);
        }
      };
      if (nj > 0) scales(0);
      for (int u = 0; u < 2 * nj; ++u) {
        const int j = u >> 1;
        bool ok = wait(raw_full + 8 * (u % 3), (uint32_t)(u / 3) & 1u, err);
        ok = ok && wait(empty + 8 * (u % NS), ((uint32_t)(u / NS) & 1u) ^ 1u, err);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (!(u & 1)) {
          float* sc = reinterpret_cast<float*>(smem + L::SC_OFF) + (j % 3) * 3 * KT;
          const bool in = (j0 + j) * KT + row < ch.kv;
          sc[row] = ks * a.c;
          sc[KT + row] = in ? lg2(vs) : 0.f;
          sc[2 * KT + row] = in ? rcp(vs) : 0.f;
          if (j + 1 < nj) scales(j + 1);
        }
        const uint32_t src = base + L::RAW_OFF + (u % 3) * RAW + row * 128;
        const uint32_t dst = base + L::RING + (uint32_t)(u % NS) * SLOT + row * 128;
#pragma unroll
        for (int cc = 0; cc < 8; ++cc) {
          const uint4 w = lds16(src + ((cc ^ sw) << 4));
          uint4 x, y;
          if (u & 1) {
            widen<PT>(w.x, x.x, x.y);
            widen<PT>(w.y, x.z, x.w);
            widen<PT>(w.z, y.x, y.y);
            widen<PT>(w.w, y.z, y.w);
          } else {
            widen<T>(w.x, x.x, x.y);
            widen<T>(w.y, x.z, x.w);
            widen<T>(w.z, y.x, y.y);
            widen<T>(w.w, y.z, y.w);
          }
          const uint32_t d = dst + (cc >> 2) * HALF;
          sts16(d + (((2 * (cc & 3)) ^ sw) << 4), x);
          sts16(d + (((2 * (cc & 3) + 1) ^ sw) << 4), y);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          arrive(raw_empty + 8 * (u % 3));
          arrive(full + 8 * (u % NS));
        }
      }
    }
    // these warps keep their few registers: their end shares no code with the others'
    __syncwarp();
    if (S > 1) {
      cluster_sync();
      cluster_sync();
    }
    fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(L::THREADS) : "memory");
    if (warp == 8) {
      fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::SOFT_REGS));
    // ------------------------------------------------ softmax: a thread per row
    const int t = warp >> 2, r = threadIdx.x & 127;   // tile, row of the tile
    const int ti = r / a.rep, i = i0 + t * a.tpt + ti;  // token within the tile, the chunk
    const bool real = ti < a.tpt && i < i0 + ntok;
    const int lim = real ? before + i + 1 : 0;        // keys that the row sees
    const int first_lim = before + i0 + t * a.tpt + 1;  // of the tile's first token, the least
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lane_off + t * 128, to = tmem + lane_off + 256 + t * 128;
    const bool active = nj > 0 && (t == 0 || two);
    float m = -INFINITY, l = 0.f;  // log2 units
    if (active) {
      for (int j = 0; j < nj; ++j) {
        if (!__all_sync(0xffffffffu, wait(s_full + 8 * t, (uint32_t)j & 1u, err))) break;
        fence_after();
        float s[128];
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) tmem_ld32(ts + 32 * cc, s + 32 * cc);
        tmem_wait_ld();
        const int key0 = (j0 + j) * KT;
        const uint32_t sc = base + L::SC_OFF + (j % 3) * 3 * KT * 4;
        if constexpr (Q8) {  // x = c k_s S + log2 v_s
#pragma unroll
          for (int e = 0; e < 128; e += 4) {
            const float4 k4 = lds16f(sc + e * 4), v4 = lds16f(sc + (KT + e) * 4);
            const float2 u = fma2(make_float2(s[e], s[e + 1]), make_float2(k4.x, k4.y), make_float2(v4.x, v4.y));
            const float2 w = fma2(make_float2(s[e + 2], s[e + 3]), make_float2(k4.z, k4.w), make_float2(v4.z, v4.w));
            s[e] = u.x, s[e + 1] = u.y, s[e + 2] = w.x, s[e + 3] = w.y;
          }
        }
        if (key0 + KT > first_lim) {
          const int vis = lim - key0;
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (e >= vis) s[e] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int e = 4; e < 124; e += 8)
#pragma unroll
          for (int x = 0; x < 4; ++x) mx[x] = max3(mx[x], s[e + x], s[e + 4 + x]);
#pragma unroll
        for (int x = 0; x < 4; ++x) mx[x] = fmaxf(mx[x], s[124 + x]);
        float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
        if (!Q8) top *= a.c;
        // the maximum in use moves only when the new one is far above it
        const bool move = top > m + (kGrow + LIFT) || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, move)) {
          const float mn = move ? top - LIFT : m;
          const float f = move && m != -INFINITY ? ex2(m - mn) : (move ? 0.f : 1.f);
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int cc = 0; cc < 8; ++cc) {
              float o[16];
              asm volatile(
                  "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                  : "=f"(o[0]), "=f"(o[1]), "=f"(o[2]), "=f"(o[3]), "=f"(o[4]), "=f"(o[5]), "=f"(o[6]), "=f"(o[7]),
                    "=f"(o[8]), "=f"(o[9]), "=f"(o[10]), "=f"(o[11]), "=f"(o[12]), "=f"(o[13]), "=f"(o[14]), "=f"(o[15])
                  : "r"(to + 16 * cc));
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              asm volatile(
                  "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(to + 16 * cc),
                  "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7]), "f"(o[8]), "f"(o[9]),
                  "f"(o[10]), "f"(o[11]), "f"(o[12]), "f"(o[13]), "f"(o[14]), "f"(o[15])
                  : "memory");
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : -m;
        // P in two halves, so that P V starts on the first
        float2 sum = make_float2(0.f, 0.f), sum2 = sum;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 64 * h; e < 64 * h + 64; e += 4) {
            float2 x, y;
            if constexpr (Q8) {
              x = add2(make_float2(s[e], s[e + 1]), make_float2(sub, sub));
              y = add2(make_float2(s[e + 2], s[e + 3]), make_float2(sub, sub));
            } else {
              x = fma2(make_float2(s[e], s[e + 1]), make_float2(a.c, a.c), make_float2(sub, sub));
              y = fma2(make_float2(s[e + 2], s[e + 3]), make_float2(a.c, a.c), make_float2(sub, sub));
            }
            x.x = ex2(x.x), x.y = ex2(x.y), y.x = ex2(y.x), y.y = ex2(y.y);
            // (rounded to the operands' type, as paged_attention.cu does)
            pk[(e & 63) / 2] = pack2<PT>(x.x, x.y);
            pk[(e & 63) / 2 + 1] = pack2<PT>(y.x, y.y);
            if constexpr (Q8) {
              const float4 r4 = lds16f(sc + (2 * KT + e) * 4);
              sum = fma2(x, make_float2(r4.x, r4.y), sum);
              sum2 = fma2(y, make_float2(r4.z, r4.w), sum2);
            } else {
              sum = add2(sum, x);
              sum2 = add2(sum2, y);
            }
          }
          tmem_st32(ts + 32 * h, pk);
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) arrive(p_full + 16 * t + 8 * h);
        }
        l += (sum.x + sum.y) + (sum2.x + sum2.y);
      }
    }
    // ------------------------------------------------ epilogue
    bool ok = !active || wait(o_full, 0, err);
    ok = __all_sync(0xffffffffu, ok);
    fence_after();
    if (S == 1) {
      const int h = g * a.rep + r % a.rep;
      T* dst = static_cast<T*>(a.out) + ((ch.q0 + i) * a.hq + h) * 128;
      bool fine = true;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // nothing seen: zeros; NaN stays
      if (active && ok) {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          float o[32];
          tmem_ld32(to + 32 * cc, o);
          tmem_wait_ld();
          if (real) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float w[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                w[x] = l == 0.f ? 0.f : o[e + x] * inv;
                fine = fine && fabsf(w[x]) < INFINITY;
              }
              reinterpret_cast<uint4*>(dst + 32 * cc + e)[0] =
                  make_uint4(pack2<T>(w[0], w[1]), pack2<T>(w[2], w[3]), pack2<T>(w[4], w[5]), pack2<T>(w[6], w[7]));
            }
          }
        }
        fine = fine && fabsf(l) < INFINITY && (Q8 || in_range<PT>(l, m));
      } else if (real) {  // a tile without any key
#pragma unroll
        for (int e = 0; e < 16; ++e) reinterpret_cast<uint4*>(dst)[e] = make_uint4(0, 0, 0, 0);
      }
      // a value that is not finite may come from a row the token does not see (0 x NaN): such
      // rows are computed again, key by key
      unsigned redo = __ballot_sync(0xffffffffu, real && active && ok && !fine);
      while (redo) {
        const int src = __ffs(redo) - 1;
        redo &= redo - 1;
        const int lm = __shfl_sync(0xffffffffu, lim, src), hh = __shfl_sync(0xffffffffu, h, src);
        const int64_t tok = __shfl_sync(0xffffffffu, ch.q0 + i, src);
        __syncwarp();
        attend_row<T, Q8>(a.p, b, g, lm, static_cast<const T*>(a.q) + (tok * a.hq + hh) * 128, a.c,
                          static_cast<T*>(a.out) + (tok * a.hq + hh) * 128);
      }
    } else {
      // ---- split over the cluster: rank z adds the parts of rows [z R, z R + R)
      const int R = 2 * QT / S, row = t * QT + r, stride = 132;
      if (!real || !active) m = -INFINITY, l = 0.f;
      sm_ml[row] = m;
      sm_ml[2 * QT + row] = l;
      __syncwarp();
      cluster_sync();  // every CTA's m and l are written, its rings are done
      float M = -INFINITY;
      for (int z = 0; z < S; ++z) M = fmaxf(M, ld_cluster(mapa(base + L::ML_OFF + row * 4, z)));
      const bool none = m == -INFINITY && !(l != 0.f);  // no key seen (a NaN score leaves l NaN)
      const float f = none ? 0.f : ex2(m - M);
      const uint32_t dst = mapa(base + (uint32_t)((rank * R + row % R) * stride) * 4, row / R);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        float o[32];
        if (active) {
          tmem_ld32(to + 32 * cc, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          if (none) st_cluster16(dst + (32 * cc + e) * 4, 0.f, 0.f, 0.f, 0.f);
          else st_cluster16(dst + (32 * cc + e) * 4, o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
        }
      }
      float Lr = 0.f;  // the row sums, by the rows' owner
      if (threadIdx.x < R) {
        const uint32_t at = base + L::ML_OFF + (rank * R + threadIdx.x) * 4;
        M = -INFINITY;
        for (int z = 0; z < S; ++z) M = fmaxf(M, ld_cluster(mapa(at, z)));
        for (int z = 0; z < S; ++z) {
          const float mz = ld_cluster(mapa(at, z)), lz = ld_cluster(mapa(at + 2 * QT * 4, z));
          if (mz != -INFINITY || lz != 0.f) Lr += lz * ex2(mz - M);
        }
        if (!Q8 && !in_range<PT>(Lr, M)) Lr = INFINITY;  // (computed again)
      }
      __syncwarp();
      cluster_sync();  // the parts have landed, and no CTA reads another's m and l any more
      if (threadIdx.x < R) sm_ml[threadIdx.x] = Lr;
      asm volatile("bar.sync 2, 256;" ::: "memory");
      for (int x = warp; x < R; x += 8) {
        const int rw = rank * R + x, tl = rw >> 7, rr = rw & 127, tk = rr / a.rep, ii = i0 + tl * a.tpt + tk;
        if (tk >= a.tpt || ii >= i0 + ntok) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < S; ++z) {
          const float4 y = lds16f(base + (uint32_t)((z * R + x) * stride + 4 * lane) * 4);
          v[0] += y.x, v[1] += y.y, v[2] += y.z, v[3] += y.w;
        }
        const float lr = sm_ml[x];
        bool fine = fabsf(lr) < INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = lr == 0.f ? 0.f : v[e] / lr;
          fine = fine && fabsf(v[e]) < INFINITY;
        }
        const int h = g * a.rep + rr % a.rep;
        const int64_t at = ((ch.q0 + ii) * a.hq + h) * 128;
        if (__all_sync(0xffffffffu, fine))
          reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at)[lane] = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        else
          attend_row<T, Q8>(a.p, b, g, before + ii + 1, static_cast<const T*>(a.q) + at, a.c, static_cast<T*>(a.out) + at);
      }
    }
    fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(L::THREADS) : "memory");
  }
}

// Key splits (CTAs of a cluster) for `units` row tiles of up to nkt key tiles: the
// fewest rounds over the SMs times the key tiles of each, plus about four tiles of
// start and end a round and two for the meeting.
int key_splits(int64_t units, int64_t nkt) {
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= 8; s *= 2) {
    if (s > 1 && nkt < 2 * s) break;
    const double rounds = (double)((units * s + sm_count() - 1) / sm_count());
    const double c = rounds * ((double)((nkt + s - 1) / s) + 4 + (s > 1 ? 2 : 0));
    if (c < cost - 1e-9) cost = c, best = s;
  }
  return best;
}

template <typename T, bool Q8>
dial_status launch(const void* q, const PagedView& p, void* out, int hq, int64_t max_kv, float c, cudaStream_t st) {
  constexpr auto kern = paged_attention_kernel<T, Q8>;
  constexpr int smem = Cfg<Q8>::BYTES;
  const int rep = hq / p.hkv, tpt = QT / rep;
  const int64_t rows = (p.n_pages * p.hkv) << p.log2_page;
  CUtensorMap qm, km, vm;
  dial_status s = make_head_map(&qm, q, p.tokens, hq, rep, tpt);
  const int box = std::min(1 << p.log2_page, KT);
  if (s == DIAL_OK) s = make_byte_map(&km, p.k, rows, Q8 ? 128 : 256, 128, box, 128);
  if (s == DIAL_OK) s = make_byte_map(&vm, p.v, rows, Q8 ? 128 : 256, 128, box, 128);
  if (s != DIAL_OK) return s;
  cudaError_t e = ensure_smem<kern>(smem);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_attention_kernel)");
  // no more tiles than the longest chunk's for every sequence, nor than the tokens fill plus
  // a broken one each
  const int64_t tiles = std::min((int64_t)p.n_seqs * ((p.max_q + 2 * tpt - 1) / (2 * tpt)), p.tokens / (2 * tpt) + p.n_seqs);
  const int64_t units = tiles * p.hkv;
  const int S = key_splits(units, (max_kv + KT - 1) / KT);
  if (units * S >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many query tiles (%lld)", (long long)units);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * S));
  cfg.blockDim = dim3(Cfg<Q8>::THREADS);
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
  const Args a{p, hq, rep, tpt, c, q, out};
  e = cudaLaunchKernelEx(&cfg, kern, qm, km, vm, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, "paged_attention_kernel");
  }
  return check_launch("paged_attention_kernel");
}

}  // namespace

dial_status launch_paged_attention_tiles(const void* q, const PagedView& p, int format, void* out, dial_dtype dt,
                                         int hq, int64_t max_kv, float c, cudaStream_t st) {
  const bool q8 = format == DIAL_KV_INT8;
  if (dt == DIAL_F16) return q8 ? launch<__half, true>(q, p, out, hq, max_kv, c, st) : launch<__half, false>(q, p, out, hq, max_kv, c, st);
  return q8 ? launch<__nv_bfloat16, true>(q, p, out, hq, max_kv, c, st)
            : launch<__nv_bfloat16, false>(q, p, out, hq, max_kv, c, st);
}

}  // namespace dial
