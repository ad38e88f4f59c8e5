// Verification of drafted tokens against the target's probabilities.
//
//   p_i = e_i / Z, e_i = exp((x_i - max x) / T), Z = sum e_i;  draft x of row r is
//   accepted if u q(x) < p(x); the token behind the last accepted one is drawn by
//   inverting the cumulative sum of w_i = max(p_i - q_i, 0) (or p_i) at u' sum w.
//
// Two launches, bound by reading the logits once (and, of one row a sequence, the
// logits again from L2 and the draft's distribution):
//   1. every row in segments of 1024, a warp each: maximum, its first index, sum of e in
//      f32, which decide the acceptances and give the log-probabilities;
//   2. a cluster of two to eight CTAs per sequence joins the segments, finds the first
//      rejected draft and draws from that row.  The index at which a cumulative sum
//      over 10^5 weights passes a random number moves with its last digits, so the
//      draw sums in f64 over exponentials good to 2^-44 (a table of 2^(j/64) and a
//      short polynomial: P. T. P. Tang, ACM TOMS 15, 1989), nine f64 operations a
//      value: every warp a run of the row, then the one run that the number falls in
//      once more, element by element.
// 32 sequences of up to 6 rows of 151936 in bf16 with the drafts' probabilities (47 MB)
// take 33 us, 9.5 of them the segments; one sequence of 4 rows takes 13.2 us, the chain of
// its steps.  The f64 pipe is busy 18 % of the draw, and with f32 exponents in its sweep the
// 32 took 0.7 us less: what binds it is the waiting from step to step (segments, acceptance,
// row, one to two meetings of the cluster, the run again), barriers before loads.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int SEG = 1024;           // a warp's piece of a row
constexpr int kStatWarps = 4;
constexpr int kDrawThreads = 512;
constexpr int kWarps = kDrawThreads / 32;
// Vectors that a thread of the draw keeps: the least that holds a warp's run of 151936 16-bit
// logits over eight CTAs (149 of 160).  Longer runs go by in pieces, and the drawn one is
// loaded again: 32 sequences of 2 rows with probabilities take 29 us at 163800 16-bit logits
// and 38 at 165000, 43 with 151936 in f32, and 52 us are 38 sequences (four CTAs each)
// where 37 take 40.  With six, two CTAs of 112 KB and their static arrays no longer fit an SM.
constexpr int HOLD = 5;
constexpr int kDrawSmem = HOLD * kDrawThreads * 32 + 64 * 32 * 8;

struct __align__(16) SegStat {
  float m, s;                // maximum, sum of exp((x - m) / T)
  unsigned long long key;    // argmax_key of the maximum (greedy sequences only)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (x - m) it of two values, two instructions
__device__ __forceinline__ float2 octaves2(float x, float y, float minus_m, float it) {
  float2 d;
  asm("{\n .reg .b64 v, m, k;\n mov.b64 v, {%2, %3};\n mov.b64 m, {%4, %4};\n mov.b64 k, {%5, %5};\n"
      " add.rn.f32x2 v, v, m;\n mul.rn.f32x2 v, v, k;\n mov.b64 {%0, %1}, v;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(x), "f"(y), "f"(minus_m), "f"(it));
  return d;
}

// Aligned 16-byte vectors over an array of `total` elements; a row's elements [lo, hi)
// need not start at one.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  // vector v, zeros behind the array's end
  static __device__ __forceinline__ uint4 load(const T* x, int64_t v, int64_t total) {
    if ((v + 1) * N <= total) return __ldg(reinterpret_cast<const uint4*>(x) + v);
    uint4 u = make_uint4(0, 0, 0, 0);
    T* h = reinterpret_cast<T*>(&u);
    for (int i = 0; i < N; ++i)
      if (v * N + i < total) h[i] = x[v * N + i];
    return u;
  }
  // its values; those outside [lo, hi) and NaN as minus infinity
  static __device__ __forceinline__ void values(uint4 u, int64_t v, int64_t lo, int64_t hi, float (&f)[N]) {
    const T* h = reinterpret_cast<const T*>(&u);
    const int a = (int)max(lo - v * N, (int64_t)0), b = (int)min(hi - v * N, (int64_t)N);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f[i] = Act<T>::to_f32(h[i]);
      if (i < a || i >= b || f[i] != f[i]) f[i] = -INFINITY;
    }
  }
};

// exp((x - m) / T) in f32 with it = log2(e) / T, x <= m; an infinite maximum takes everything
__device__ __forceinline__ float weight32(float x, float m, float it) { return x == m ? 1.f : ex2((x - m) * it); }
__device__ __forceinline__ float log2e_over(float temp) { return temp > 0.f ? __fdiv_rn(1.442695041f, temp) : 1.442695041f; }

struct Rows {
  int64_t q0, q1;
};
__device__ __forceinline__ Rows rows_of(const VerifyArgs& a, int b, bool report) {
  const int64_t s0 = a.q_start[b], s1 = a.q_start[b + 1];
  const int64_t q0 = s0 < 0 ? 0 : (s0 > a.rows ? a.rows : s0);
  int64_t q1 = s1 < q0 ? q0 : (s1 > a.rows ? a.rows : s1);
  if (report && (q0 != s0 || q1 != s1 || q1 - q0 > a.max_q)) flag_invalid(a.err);
  if (q1 - q0 > a.max_q) q1 = q0 + a.max_q;
  return {q0, q1};
}

// ------------------------------------------------------------------ 1. the rows' segments
// Four instructions and an ex2 a value: the ex2 rate (16 a clock and SM) is what is
// near the bytes' time.
template <typename T>
__global__ void __launch_bounds__(kStatWarps * 32) verify_stats_kernel(VerifyArgs a, SegStat* __restrict__ stat, int nseg) {
  pdl_begin();
  constexpr int N = Vec<T>::N, PER = SEG / 32 / N;
  const int64_t w = (int64_t)blockIdx.x * kStatWarps + (threadIdx.x >> 5);
  if (w >= a.rows * nseg) return;
  const int64_t row = w / nseg, total = a.rows * a.vocab;
  const int lane = threadIdx.x & 31;
  // segments start at the row's own aligned vectors: the first has the row's first elements,
  // the last one more vector if the row ends inside it
  const int64_t lo = row * a.vocab, hi = lo + a.vocab;
  const int64_t v0 = lo / N + (w - row * nseg) * (SEG / N);
  const T* x = static_cast<const T*>(a.logits);
  uint4 u[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) u[k] = Vec<T>::load(x, v0 + k * 32 + lane, total);
  const int b = seq_of_token(a.q_start, a.n_seqs, row);
  if (b >= a.n_seqs) return;
  const float temp = a.temperature[b], it = log2e_over(temp);
  float f[PER][N], m = -INFINITY;
  const bool inside = v0 * N >= lo && (v0 + SEG / N) * N <= hi;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (inside) {
      const T* h = reinterpret_cast<const T*>(&u[k]);
#pragma unroll
      for (int i = 0; i < N; ++i) f[k][i] = Act<T>::to_f32(h[i]);
    } else {
      Vec<T>::values(u[k], v0 + k * 32 + lane, lo, hi, f[k]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, f[k][i]);
  }
  const float mine = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = 0.f;
  // (the difference first: x it - m it would be off by 2^-24 |m| / T octaves)
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = octaves2(f[k][i], f[k][i + 1], -m, it);
      s += ex2(y.x), s += ex2(y.y);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (!(s < INFINITY)) {  // NaN logits, an infinite maximum, or none
    s = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (f[k][i] > -INFINITY) s += weight32(f[k][i], m, it);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  unsigned long long key = 0ull;
  if (!(temp > 0.f)) {  // greedy: the first index of the maximum
    if (mine == m) {
      int at = 0;
#pragma unroll
      for (int k = PER - 1; k >= 0; --k)
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
          if (f[k][i] == m) at = (k * 32 + lane) * N + i;
      key = argmax_key(m, v0 * N + at - lo);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  }
  if (lane == 0) stat[w] = {m, s, key};
}

// ------------------------------------------------------------------ 2. acceptance and the draw
__device__ const double kPow2[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

// exp((x - m) / T) up to a factor that all of a row share, to 2^-44, in nine f64
// operations (a cubic, good to 2^-34, leaves 2^-11 of a weight max(p - q, 0) of 2^-23 p).  Values 672 T or more below the maximum, minus infinity and NaN give what
// `least` gives, 2^-970 up to `least`'s own rounding, 32 T or 46 octaves where T is 2^-29 |m|
// (kSharp: below it they are not asked for).  No sum feels that, and kNone, above 2^30 times
// 2^-923, tells it from a weight: a run's sum above kNone is one.  The run has fewer than 2^24
// vectors, so one of them is above kNoneVec then, and of its at most eight elements one is above
// kNoneOne, still 2^6 times what `least` gives.  Every lane has a copy of the table in its own
// banks: entry j of lane l at table[32 j + l].
constexpr double kNone = 0x1p-890, kNoneVec = 0x1p-914, kNoneOne = 0x1p-917;
// A row whose T is below kSharp |m|: the next f32 below m is 32 T or more away and weighs
// less than 2^-46, so that the maximum takes everything.
constexpr float kSharp = 0x1p-29f;
struct Exp {
  const double* table;  // 2^(j / 64), this lane's
  double k, c;          // 64 log2(e) / T, minus m times that
  float least;
  __device__ __forceinline__ Exp(const double* t, float m, float temp, double k64)
      : table(t + (threadIdx.x & 31)), k(k64), c(-(double)m * k64), least(fmaxf(m - 672.f * temp, -3e38f)) {}
  __device__ __forceinline__ double operator()(float x) const {
    const double y = fma((double)fmaxf(x, least), k, c);
    const double t = y + 6755399441055744.0;            // 1.5 * 2^52: the integer in the low word
    const int n = __double2loint(t);
    const double r = y - (t - 6755399441055744.0);
    double p = 5.732851688640402e-10;                   // (ln2 / 64)^j / j!
    p = fma(p, r, 2.1173137155464774e-07);
    p = fma(p, r, 5.864904955056169e-05);
    p = fma(p, r, 0.010830424696249145);
    const double e = table[(n & 63) * 32];
    const double v = fma(e, p * r, e);
    return __hiloint2double(__double2hiint(v) + (n >> 6) * (1 << 20), __double2loint(v));
  }
};

__device__ __forceinline__ uint32_t map_shared(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The runs' sums meet: every warp puts its own into sum[] of every CTA of the cluster (a
// buffer that the call before last used); afterwards every warp knows the total, the run
// that `u` times it falls in and the sum before that run (the last run of any weight,
// should rounding leave none).  `three`: the sums are mine = sum of e, a and q, the weights
// a - z q with z the total of e.
template <int CL>
__device__ __forceinline__ double meet(double* sum, int rank, bool three, double mine, double a, double q, double& z,
                                       double u, int& run, double& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int ALL = CL * kWarps;
  if (lane < CL) {
    const uint32_t at = map_shared(sum + rank * kWarps + warp, lane);
    st_cluster_f64(at, mine);
    if (three) st_cluster_f64(at + ALL * 8, a), st_cluster_f64(at + 2 * ALL * 8, q);
  }
  __syncwarp();
  cluster_sync();
  constexpr int PER = ALL / 32;
  double v[PER], s = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = sum[lane * PER + i];
    s += v[i];
  }
  if (three) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    z = s;
    s = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = fmax(fma(-z, sum[2 * ALL + lane * PER + i], sum[ALL + lane * PER + i]), 0.0);
      s += v[i];
    }
  }
  double pre = s;  // inclusive prefix over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += y;
  }
  const double total = __shfl_sync(0xffffffffu, pre, 31), at = u * total;
  double cum = pre - s;
  int hit = CL * kWarps, last = -1;
  double hit_before = 0.0, last_before = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (v[i] > kNone) last = lane * PER + i, last_before = cum;
    if (hit == CL * kWarps && v[i] > kNone && cum + v[i] > at) hit = lane * PER + i, hit_before = cum;
    cum += v[i];
  }
  const unsigned some = __ballot_sync(0xffffffffu, hit < CL * kWarps), any = __ballot_sync(0xffffffffu, last >= 0);
  if (some) {
    const int l = __ffs(some) - 1;
    run = __shfl_sync(0xffffffffu, hit, l);
    before = __shfl_sync(0xffffffffu, hit_before, l);
  } else {
    const int l = any ? 31 - __clz(any) : 0;
    run = __shfl_sync(0xffffffffu, last, l);
    before = __shfl_sync(0xffffffffu, last_before, l);
  }
  return total;
}

template <typename T, int CL, int PER_SM>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(kDrawThreads, PER_SM)
    verify_draw_kernel(VerifyArgs a, const SegStat* __restrict__ stat, int nseg) {
  constexpr int N = Vec<T>::N;
  __shared__ __align__(16) double sum[2][3 * CL * kWarps];
  extern __shared__ __align__(16) uint8_t draw_smem[];
  uint4(*held)[kDrawThreads] = reinterpret_cast<uint4(*)[kDrawThreads]>(draw_smem);  // this thread's vectors
  double(*part)[kDrawThreads] = reinterpret_cast<double(*)[kDrawThreads]>(draw_smem + HOLD * kDrawThreads * 16);  // their sums
  double(*partq)[kDrawThreads] = reinterpret_cast<double(*)[kDrawThreads]>(draw_smem + HOLD * kDrawThreads * 24);
  double* table = reinterpret_cast<double*>(draw_smem + HOLD * kDrawThreads * 32);  // [64][32]
  __shared__ float row_m[kWarps], row_z[kWarps], row_x[kWarps];
  __shared__ int row_top[kWarps], row_ok[kWarps], row_draft[kWarps];
  pdl_trigger();
  cluster_arrive();  // every CTA runs before another writes to it
  for (int i = threadIdx.x; i < 64 * 32; i += kDrawThreads) table[i] = kPow2[i / 32];
  pdl_wait();
  const int b = blockIdx.x / CL, rank = blockIdx.x % CL;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Rows rw = rows_of(a, b, rank == 0 && threadIdx.x == 0);
  const int64_t V = a.vocab, total = a.rows * V;
  const T* x = static_cast<const T*>(a.logits);
  const float tb = a.temperature[b], temp = tb > 1e30f ? 1e30f : tb, it = log2e_over(temp);
  const float ut = a.sample_u[b];
  const bool greedy = !(temp > 0.f);
  const double k64 = greedy ? 0.0 : 92.332482616893656 / (double)temp;  // 64 log2(e) / T
  if (rw.q0 == rw.q1) {
    if (rank == 0 && threadIdx.x == 0) a.n_out[b] = 0;
    __syncwarp();
    cluster_wait();
    return;  // the whole cluster: no rows
  }

  // ---- acceptance, a warp per row
  int64_t stop = rw.q1 - 1;
  float m = 0.f, Z = 0.f;
  int top = 0, draft = -1;
  bool rejected = false;
  auto log_p = [&](float v, float mr, float z) -> float {  // log of exp((v - mr) / T) / z
    if (z == 0.f || !(v > -INFINITY) || (mr == INFINITY && v != mr)) return -INFINITY;
    return (v == mr ? 0.f : greedy ? v - mr : __fdiv_rn(v - mr, temp)) - logf(z);
  };
  for (int64_t r0 = rw.q0; r0 < rw.q1; r0 += kWarps) {
    const int64_t r = r0 + warp;
    __syncthreads();
    if (r < rw.q1) {
      const bool judge = r + 1 < rw.q1;
      const int d = judge ? a.ids[r + 1] : -1;
      const bool in = d >= 0 && d < V;
      const float xd = in ? Act<T>::to_f32(x[r * V + d]) : -INFINITY;
      const float qd = in && a.probs ? a.probs[r * V + d] : 1.f, ua = judge ? a.accept_u[r] : 0.f;
      float mr = -INFINITY, z = 0.f;
      unsigned long long key = 0ull;
#pragma unroll 4
      for (int i = lane; i < nseg; i += 32) {
        const SegStat s = stat[r * nseg + i];
        const float mn = fmaxf(mr, s.m);
        z = z * weight32(mr, mn, it) + s.s * weight32(s.m, mn, it);
        mr = mn;
        key = max(key, s.key);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, mr, o), zo = __shfl_xor_sync(0xffffffffu, z, o), mn = fmaxf(mr, mo);
        z = z * weight32(mr, mn, it) + zo * weight32(mo, mn, it);
        mr = mn;
        key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
      }
      int t = (int)(0xFFFFFFFFu - (uint32_t)key);
      t = z == 0.f || t < 0 || t >= V ? 0 : t;
      const bool ok = in && (greedy ? d == t : xd > -INFINITY && z > 0.f && (double)ua * qd * z < weight32(xd, mr, it));
      if (lane == 0) row_m[warp] = mr, row_z[warp] = z, row_x[warp] = xd, row_top[warp] = t, row_ok[warp] = ok, row_draft[warp] = d;
    }
    __syncthreads();
    const int n = (int)min((int64_t)kWarps, rw.q1 - r0);
    const unsigned good = __ballot_sync(0xffffffffu, lane < n && row_ok[lane & (kWarps - 1)]);
    const int k = good == 0xffffffffu ? 32 : __ffs(~good) - 1;  // the accepted ones in front
    if (rank == 0 && threadIdx.x < k) {
      a.out_ids[r0 + threadIdx.x] = row_draft[threadIdx.x];
      if (a.logprobs) a.logprobs[r0 + threadIdx.x] = log_p(row_x[threadIdx.x], row_m[threadIdx.x], row_z[threadIdx.x]);
    }
    if (k < n) {  // row r0 + k ends the output: a rejected draft, or no draft left
      stop = r0 + k;
      rejected = stop + 1 < rw.q1;
      m = row_m[k], Z = row_z[k], top = row_top[k], draft = row_draft[k];
      break;
    }
  }
  if (rank == 0) {
    if (threadIdx.x == 0) a.n_out[b] = (int)(stop - rw.q0 + 1);
    for (int64_t i = stop + 1 + threadIdx.x; i < rw.q1; i += kDrawThreads) {
      a.out_ids[i] = -1;
      if (a.logprobs) a.logprobs[i] = 0.f;
    }
  }
  auto tell = [&](int token, float v) {
    a.out_ids[stop] = token;
    if (a.logprobs) a.logprobs[stop] = log_p(v, m, Z);
  };
  if (greedy || Z == 0.f) {
    if (rank == 0 && threadIdx.x == 0) tell(top, m);
    __syncwarp();
    cluster_wait();
    return;  // the whole cluster: it decides the same everywhere
  }

  // ---- the draw from row `stop`: run w of CL * kWarps, in whole vectors
  const bool sharp = temp < kSharp * fabsf(m);  // (an infinite one too) weights 1 at the maximum
  const Exp ex(table, sharp ? 0.f : m, temp, k64);
  // (vectors counted from the row's first, which like its last may hold other rows' values)
  const int64_t lo = stop * V, hi = lo + V, v0 = lo / N;
  const int nv = (int)((hi + N - 1) / N - v0), per = (nv + CL * kWarps - 1) / (CL * kWarps);
  const int a0 = min(nv, (rank * kWarps + warp) * per), a1 = min(nv, a0 + per);
  const uint4* xv = reinterpret_cast<const uint4*>(x) + v0;
  const float* qv = a.probs + v0 * N;
  const bool cut = (v0 + nv) * N > total;  // the last vector passes the array's end
  const int to_draft = draft >= 0 && draft < V ? (int)(lo + draft - v0 * N) : -1;
  double z64 = 0.0;
  const double z0 = (double)Z;
  // 0: all of p; 1: p without the draft; 3: max(p - q, 0) Z = max(e - q Z, 0) in one pass, by
  // the sums of e and q where e > q z0, z0 being Z as the segments gave it in f32: off by
  // 2^-23 of it or so, by 2^-17 at most (an exponent of 17 octaves has three roundings of
  // 2^-24 of it, ex2 one of 2^-22, and a sum of 2^18 values goes through some 40 additions).
  // Nothing else depends on z0, and a value on the wrong side of it has a weight of
  // |e - q Z| <= q |z0 - Z|, all of them together |z0 - Z|.  Both are known after the pass:
  // where what is left of p is not 2^16 times that (or below 2^-12 of p, which the difference
  // of two sums would feel) 2 follows: the same with Z in f64 throughout.
  int mode = !rejected ? 0 : (a.probs ? 3 : 1);
  auto values = [&](uint4 u, int v, float (&f)[N]) {
    if (v == 0 || v == nv - 1) {
      Vec<T>::values(u, v0 + v, lo, hi, f);
    } else {
      const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = Act<T>::to_f32(h[i]);
    }
    if (sharp) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = f[i] == m ? 0.f : -INFINITY;
    }
    if (mode == 1 && v == to_draft / N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (v * N + i == to_draft) f[i] = -INFINITY;
    }
  };
  auto draft_probs = [&](int v, float (&q)[N]) {
    if (!cut || v < nv - 1) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 y = __ldg(reinterpret_cast<const float4*>(qv + v * N + i));
        q[i] = y.x, q[i + 1] = y.y, q[i + 2] = y.z, q[i + 3] = y.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = (v0 + v) * N + i < total ? qv[v * N + i] : 0.f;
    }
    if (v == 0 || v == nv - 1) {  // other rows' values, whatever they are, are none of this row's
      const int64_t e = (v0 + v) * N;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e + i < lo || e + i >= hi) q[i] = 0.f;
    }
  };
  auto weight1 = [&](int64_t e) {  // of one element of the row
    float f = Act<T>::to_f32(x[e]);
    if (sharp) f = f == m ? 0.f : -INFINITY;
    if (mode == 1 && e - lo == draft) f = -INFINITY;
    const double w = ex(f);
    if (mode < 2) return w;
    const double q = (double)a.probs[e];
    return mode == 3 && !(fma(-q, z0, w) > 0.0) ? 0.0 : fmax(fma(-q, z64, w), 0.0);
  };
  if (mode == 3)  // the draft's weights of this run, wanted soon
    for (int e = a0 * N + 32 * lane; e < a1 * N && v0 * N + e < total; e += 32 * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(qv + e));
  __syncwarp();
  cluster_wait();
  const double u = (double)ut;
  const bool single = per <= 32 * HOLD;  // all sums of the run are kept
  bool loaded = false;
  int run = -1, buf = 0, token = -1;
  double before = 0.0, all = 0.0, at = 0.0;
  // passes over the run: for Z, for the weights, and for the place of `at`.  The loops stay
  // rolled: code that runs once or twice a launch waits for its instructions.
  for (;;) {
    const bool locate = run >= 0;
    double mine = 0.0, mina = 0.0, minq = 0.0, cum = before;
    bool found = false;
#pragma unroll 1
    for (int c0 = a0; c0 < a1 && !found; c0 += 32 * HOLD) {
      if (!locate || !single) {
        if (!single || !loaded) {  // all in flight at once; each thread reads back its own
#pragma unroll
          for (int k = 0; k < HOLD; ++k) {
            const int v = c0 + 32 * k + lane;
            if (v < a1 && !(cut && v == nv - 1))
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&held[k][threadIdx.x])),
                           "l"(xv + v)
                           : "memory");
            else if (v < a1)
              held[k][threadIdx.x] = Vec<T>::load(x, v0 + v, total);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          loaded = true;
        }
#pragma unroll 1
        for (int k = 0; k < HOLD; ++k) {
          const int v = c0 + 32 * k + lane;
          double s = 0.0, sa = 0.0, sq = 0.0;
          if (v < a1) {
            float f[N];
            values(held[k][threadIdx.x], v, f);
            if (mode >= 2) {  // (outside the row e is nothing and q is 0)
              float q[N];
              draft_probs(v, q);
              const double z = mode == 3 ? z0 : z64;
#pragma unroll
              for (int i = 0; i < N; ++i) {
                const double w = ex(f[i]), qd = (double)q[i], d = fma(-qd, z, w);
                const bool over = __double2hiint(d) >= 0;
                s += mode == 3 ? w : (over ? d : 0.0);
                sa += over ? w : 0.0;
                sq += over ? qd : 0.0;
              }
            } else {
              double s2 = 0.0;
#pragma unroll
              for (int i = 0; i < N; i += 2) s += ex(f[i]), s2 += ex(f[i + 1]);
              s += s2;
            }
          }
          part[k][threadIdx.x] = mode == 3 ? sa : s;
          partq[k][threadIdx.x] = sq;
          mine += s;
          mina += sa;
          minq += sq;
        }
      }
      if (!locate) continue;
      // the vector in which the cumulative sum passes `at`, or the last of any weight
      int vec = -1;
      double start = 0.0;
#pragma unroll 1
      for (int k = 0; k < HOLD && !found; ++k) {
        double s = part[k][threadIdx.x];
        if (mode == 3) s = fmax(fma(-z64, partq[k][threadIdx.x], s), 0.0);
        double pre = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, pre, o);
          if (lane >= o) pre += y;
        }
        const unsigned some = __ballot_sync(0xffffffffu, s > kNoneVec && cum + pre > at);
        const unsigned any = __ballot_sync(0xffffffffu, s > kNoneVec);
        if (any) {
          const int l = some ? __ffs(some) - 1 : 31 - __clz(any);
          vec = c0 + 32 * k + l;
          start = cum + __shfl_sync(0xffffffffu, pre - s, l);
          found = some != 0;
        }
        cum += __shfl_sync(0xffffffffu, pre, 31);
      }
      if (vec >= 0) {  // its element, a lane each
        const int64_t e = (v0 + vec) * N + lane;
        const double w = lane < N && e >= lo && e < hi ? weight1(e) : 0.0;
        double pre = w;
#pragma unroll
        for (int o = 1; o < N; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, pre, o);
          if (lane >= o) pre += y;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > kNoneOne && start + pre > at);
        const unsigned any = __ballot_sync(0xffffffffu, w > kNoneOne);
        if (any) token = (int)((v0 + vec) * N + (some ? __ffs(some) - 1 : 31 - __clz(any)) - lo);
      }
    }
    if (locate) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
      if (mode == 3) mina += __shfl_xor_sync(0xffffffffu, mina, o), minq += __shfl_xor_sync(0xffffffffu, minq, o);
    }
    int r;
    all = meet<CL>(sum[buf], rank, mode == 3, mine, mina, minq, z64, u, r, before);
    buf ^= 1;
    if (mode == 3 && !(all > fmax(z64 * 0x1p-12, fabs(z64 - z0) * 0x1p16))) {
      mode = 2;
    } else if (mode && mode != 3 && !(all > kNone)) {
      mode = 0;  // nothing left of it: from p
    } else {
      if (r != rank * kWarps + warp) break;
      run = r;
      at = u * all;
    }
  }
  if (run >= 0) {
    // (sums of max(p - q, 0) that rounding alone raised above zero leave no element: the maximum)
    for (int64_t e = lane; token < 0 && e - lane < V; e += 32) {
      const unsigned at_max = __ballot_sync(0xffffffffu, e < V && Act<T>::to_f32(x[lo + min(e, V - 1)]) == m);
      if (at_max) token = (int)(e - lane) + __ffs(at_max) - 1;
    }
    if (lane == 0) tell(token, Act<T>::to_f32(x[lo + token]));
  }
  __syncwarp();
  cluster_sync();  // nobody leaves while another reads its sums
}

// a row's vectors, from the one that holds its first element on, in pieces of SEG
int64_t segments(int64_t vocab) { return (vocab + 7 + SEG - 1) / SEG; }

}  // namespace

size_t verify_workspace_bytes(int64_t rows, int64_t vocab) {
  return (size_t)(rows * segments(vocab)) * sizeof(SegStat);
}

template <typename T, int CL, int PER_SM>
static dial_status launch_draw(const VerifyArgs& a, const SegStat* stat, int nseg, cudaStream_t st) {
  const cudaError_t e = ensure_smem<verify_draw_kernel<T, CL, PER_SM>>(kDrawSmem);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(verify_draw_kernel)");
  return launch_pdl("verify_draw_kernel", verify_draw_kernel<T, CL, PER_SM>, dim3((unsigned)(a.n_seqs * CL)), dim3(kDrawThreads),
                    kDrawSmem, st, a, stat, nseg);
}

template <typename T>
static dial_status verify_t(const VerifyArgs& a, void* ws, cudaStream_t st) {
  const int64_t nseg = segments(a.vocab), blocks = (a.rows * nseg + kStatWarps - 1) / kStatWarps;
  SegStat* stat = static_cast<SegStat*>(ws);
  if (blocks >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many rows (%lld)", (long long)a.rows);
  const dial_status s = launch_pdl("verify_stats_kernel", verify_stats_kernel<T>, dim3((unsigned)blocks),
                                   dim3(kStatWarps * 32), 0, st, a, stat, (int)nseg);
  if (s != DIAL_OK) return s;
  // CTAs per sequence: eight (the portable cluster) while they have an SM each or share it
  // with one other (64 registers then: 12.7 -> 14.0 us for one sequence, but 49 -> 39 us for
  // 32 against four CTAs each), then fewer
  const int64_t ctas = 8 * (int64_t)a.n_seqs, sms = sm_count();
  return ctas <= sms       ? launch_draw<T, 8, 1>(a, stat, (int)nseg, st)
         : ctas <= 2 * sms ? launch_draw<T, 8, 2>(a, stat, (int)nseg, st)
         : ctas <= 4 * sms ? launch_draw<T, 4, 2>(a, stat, (int)nseg, st)
                           : launch_draw<T, 2, 2>(a, stat, (int)nseg, st);
}

dial_status launch_verify(const VerifyArgs& a, dial_dtype dt, void* ws, cudaStream_t st) {
  return dt == DIAL_F16 ? verify_t<__half>(a, ws, st) : dt == DIAL_BF16 ? verify_t<__nv_bfloat16>(a, ws, st) : verify_t<float>(a, ws, st);
}

}  // namespace dial
