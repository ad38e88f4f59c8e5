// Verification of drafted tokens against the target's probabilities.
//
//   p_i = e_i / Z, e_i = exp((x_i - max x) / T), Z = sum e_i;  draft x of row r is
//   accepted if u q(x) < p(x); the token behind the last accepted one is drawn by
//   inverting the cumulative sum of w_i = max(p_i - q_i, 0) (or p_i) at u' sum w.
//
// Two launches, bound by reading the logits once (and, of one row a sequence, the
// logits again from L2 and the draft's distribution):
//   1. every row in segments of 4096: maximum, first index of it, sum of e in f32,
//      which decide the acceptances and give the log-probabilities;
//   2. a cluster of eight CTAs per sequence joins the segments, finds the first
//      rejected draft and draws from that row.  The index at which a cumulative sum
//      over 10^5 weights passes a random number moves with its last digits, so the
//      draw sums in f64 over exponentials good to 2^-45 (a table of 2^(j/64) and a
//      short polynomial: P. T. P. Tang, ACM TOMS 15, 1989), eleven f64 operations a
//      value: every warp a run of the row, then the one run that the number falls in
//      once more, element by element.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int SEG = 4096;
constexpr int kStatThreads = 256;
constexpr int kDrawThreads = 512;
constexpr int kWarps = kDrawThreads / 32;
constexpr int kCluster = 8;

struct __align__(16) SegStat {
  float m, s;                // maximum, sum of exp((x - m) / T)
  unsigned long long key;    // argmax_key of the maximum
};

// The aligned vectors that hold elements [lo, hi) of an array of `total` elements;
// values outside [lo, hi) and NaN come as minus infinity.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void load(const T* x, int64_t v, int64_t lo, int64_t hi, int64_t total, float (&f)[N]) {
    const int64_t e0 = v * N;
    if (e0 + N <= total) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(x) + v);
      const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = Act<T>::to_f32(h[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = e0 + i < total ? Act<T>::to_f32(x[e0 + i]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (e0 + i < lo || e0 + i >= hi || f[i] != f[i]) f[i] = -INFINITY;
  }
};

// exp((x - m) / T) in f32 with it = log2(e) / T, split so that the exponent is good to
// an ulp of the result; an infinite maximum takes everything.
__device__ __forceinline__ float weight32(float x, float m, float it, float it_lo) {
  if (m == INFINITY) return x == m ? 1.f : 0.f;
  if (x == -INFINITY) return 0.f;
  const float d = x - m, h = d * it, lo = fmaf(d, it, -h) + d * it_lo;
  return exp2f(h) * fmaf(lo, 0.6931472f, 1.f);
}

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
template <typename T>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(VerifyArgs a, SegStat* __restrict__ stat) {
  pdl_begin();
  constexpr int N = Vec<T>::N, PER = SEG / kStatThreads / N;
  __shared__ float red[kStatThreads / 32];
  __shared__ unsigned long long kred[kStatThreads / 32];
  const int nseg = (int)((a.vocab + SEG - 1) / SEG);
  const int64_t row = blockIdx.x / nseg, total = a.rows * a.vocab;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b = 0;  // the row's sequence
  for (int i = 0; i < a.n_seqs; i += 32) {
    const bool past = i + lane < a.n_seqs && __ldg(a.q_start + i + lane + 1) <= row;
    const int c = __popc(__ballot_sync(0xffffffffu, past));
    b += c;
    if (c < 32) break;
  }
  if (b >= a.n_seqs) return;
  const int64_t r0 = row * a.vocab, lo = r0 + (int64_t)(blockIdx.x % nseg) * SEG;
  const int64_t hi = min(lo + SEG, r0 + a.vocab);
  const T* x = static_cast<const T*>(a.logits);
  float f[PER + 1][N];  // a segment that starts inside a vector reaches into one more
  const int64_t v0 = lo / N;
#pragma unroll
  for (int k = 0; k < PER; ++k) Vec<T>::load(x, v0 + k * kStatThreads + threadIdx.x, lo, hi, total, f[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) f[PER][i] = -INFINITY;
  const int64_t extra = v0 + SEG / N;
  if (threadIdx.x == 0 && extra * N < hi) Vec<T>::load(x, extra, lo, hi, total, f[PER]);
  const float temp = a.temperature[b];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k <= PER; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, f[k][i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kStatThreads / 32; ++w) m = fmaxf(m, red[w]);
  const double itd = (temp > 0.f ? 1.0 / (double)temp : 1.0) * 1.4426950408889634;
  const float it = (float)itd, it_lo = (float)(itd - (double)it);
  float s = 0.f;
  unsigned long long key = 0ull;
#pragma unroll
  for (int k = 0; k <= PER; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s += weight32(f[k][i], m, it, it_lo);
      if (f[k][i] == m) {
        const int64_t e = (k < PER ? (v0 + k * kStatThreads + threadIdx.x) : extra) * N + i;
        if (e >= lo && e < hi) key = max(key, argmax_key(m, e - r0));
      }
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  }
  __syncthreads();
  if (lane == 0) red[warp] = s, kred[warp] = key;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < kStatThreads / 32; ++w) s += red[w], key = max(key, kred[w]);
    stat[blockIdx.x] = {m, s, key};
  }
}

// ------------------------------------------------------------------ 2. acceptance and the draw
struct Exp {
  const double* table;  // 2^(j / 64)
  double m, k;          // maximum, log2(e) / T
  float mf;
  __device__ __forceinline__ double operator()(float x) const {
    if (mf == INFINITY) return x == mf ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    const double y = ((double)x - m) * k;
    if (y < -1000.0) return 0.0;
    const double t = fma(y, 64.0, 6755399441055744.0);  // 1.5 * 2^52: the integer in the low word
    const int n = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -1.0 / 64, y);
    double p = 0.00961812910762847716;                  // ln2^j / j!
    p = fma(p, r, 0.05550410866482157995);
    p = fma(p, r, 0.24022650695910071233);
    p = fma(p, r, 0.69314718055994530942);
    const double e = table[n & 63];
    const double v = fma(e, p * r, e);
    return __hiloint2double(__double2hiint(v) + (n >> 6) * (1 << 20), __double2loint(v));
  }
};

__device__ __forceinline__ uint32_t map_shared(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The runs' sums meet: sum[w] of every CTA of the cluster; afterwards every warp
// knows the total and, as a pair, the run that `u` times it falls in and the sum
// before that run (the last run of any weight, should rounding leave none).
__device__ __forceinline__ double meet(double* sum, double mine, double u, int& run, double& before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sum[warp] = mine;
  cluster_sync();
  constexpr int PER = kCluster * kWarps / 32;
  double v[PER], s = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = lane * PER + i;
    v[i] = ld_cluster_f64(map_shared(sum + r % kWarps, r / kWarps));
    s += v[i];
  }
  double pre = s;  // inclusive prefix over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += y;
  }
  const double total = __shfl_sync(0xffffffffu, pre, 31), at = u * total;
  double cum = pre - s;
  int hit = kCluster * kWarps, last = -1;
  double hit_before = 0.0, last_before = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (v[i] > 0.0) last = lane * PER + i, last_before = cum;
    if (hit == kCluster * kWarps && v[i] > 0.0 && cum + v[i] > at) hit = lane * PER + i, hit_before = cum;
    cum += v[i];
  }
  const unsigned some = __ballot_sync(0xffffffffu, hit < kCluster * kWarps), any = __ballot_sync(0xffffffffu, last >= 0);
  if (some) {
    const int l = __ffs(some) - 1;
    run = __shfl_sync(0xffffffffu, hit, l);
    before = __shfl_sync(0xffffffffu, hit_before, l);
  } else {
    const int l = any ? 31 - __clz(any) : 0;
    run = __shfl_sync(0xffffffffu, last, l);
    before = __shfl_sync(0xffffffffu, last_before, l);
  }
  cluster_sync();  // the sums may be written again
  return total;
}

template <typename T>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kDrawThreads)
    verify_draw_kernel(VerifyArgs a, const SegStat* __restrict__ stat, int nseg) {
  pdl_begin();
  constexpr int N = Vec<T>::N;
  __shared__ double table[64], sum[kWarps];
  __shared__ float row_m[kWarps];
  __shared__ double row_z[kWarps];
  __shared__ int row_top[kWarps], row_ok[kWarps];
  const int b = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Rows rw = rows_of(a, b, rank == 0 && threadIdx.x == 0);
  const int64_t V = a.vocab, total = a.rows * V;
  const T* x = static_cast<const T*>(a.logits);
  const float temp = a.temperature[b];
  const bool greedy = !(temp > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)temp;
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64);
  if (rw.q0 == rw.q1) {
    if (rank == 0 && threadIdx.x == 0) a.n_out[b] = 0;
    return;  // the whole cluster: no rows
  }

  // ---- acceptance, a warp per row, sixteen rows at a time
  int64_t stop = rw.q1 - 1;
  float m = 0.f;
  double Z = 0.0;
  int top = 0;
  bool rejected = false;
  for (int64_t r0 = rw.q0; r0 < rw.q1; r0 += kWarps) {
    const int64_t r = r0 + warp;
    __syncthreads();
    if (r < rw.q1) {
      float mr = -INFINITY;
      unsigned long long key = 0ull;
      for (int i = lane; i < nseg; i += 32) {
        const SegStat s = stat[r * nseg + i];
        mr = fmaxf(mr, s.m);
        key = max(key, s.key);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        mr = fmaxf(mr, __shfl_xor_sync(0xffffffffu, mr, o));
        key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
      }
      double z = 0.0;
      for (int i = lane; i < nseg; i += 32) {
        const SegStat s = stat[r * nseg + i];
        if (s.m == mr) z += s.s;
        else if (mr != INFINITY && s.m != -INFINITY) z += (double)s.s * exp(((double)s.m - (double)mr) * inv_t);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      int t = (int)(0xFFFFFFFFu - (uint32_t)key);
      t = z == 0.0 ? 0 : (t < 0 || t >= V ? 0 : t);
      bool ok = false;
      if (r + 1 < rw.q1) {
        const int draft = a.ids[r + 1];
        ok = draft >= 0 && draft < V;
        if (ok && greedy) {
          ok = draft == t;
        } else if (ok) {
          const float xd = Act<T>::to_f32(x[r * V + draft]);
          const double q = a.probs ? (double)a.probs[r * V + draft] : 1.0;
          const double e = xd == mr ? (mr == -INFINITY ? 0.0 : 1.0)
                                    : (mr == INFINITY || !(xd > -INFINITY) ? 0.0 : exp(((double)xd - (double)mr) * inv_t));
          ok = (double)a.accept_u[r] * q * z < e;
        }
      }
      if (lane == 0) row_m[warp] = mr, row_z[warp] = z, row_top[warp] = t, row_ok[warp] = ok;
    }
    __syncthreads();
    const int n = (int)min((int64_t)kWarps, rw.q1 - r0);
    int k = 0;
    while (k < n && row_ok[k]) ++k;
    const bool done = k < n;  // row r0 + k is the last of the output: a rejected draft, or no draft left
    auto log_p = [&](int w, float v) -> float {
      if (row_z[w] == 0.0 || v != v) return -INFINITY;
      if (v == row_m[w]) return (float)-log(row_z[w]);
      return row_m[w] == INFINITY ? -INFINITY : (float)(((double)v - (double)row_m[w]) * inv_t - log(row_z[w]));
    };
    if (rank == 0 && threadIdx.x < k) {
      const int64_t q = r0 + threadIdx.x;
      const int draft = a.ids[q + 1];
      a.out_ids[q] = draft;
      if (a.logprobs) a.logprobs[q] = log_p(threadIdx.x, Act<T>::to_f32(x[q * V + draft]));
    }
    if (done) {
      stop = r0 + k;
      rejected = stop + 1 < rw.q1;
      m = row_m[k], Z = row_z[k], top = row_top[k];
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
    if (!a.logprobs) return;
    float lp = -INFINITY;
    if (Z != 0.0 && v == m) lp = (float)-log(Z);
    else if (Z != 0.0 && m != INFINITY && v > -INFINITY) lp = (float)(((double)v - (double)m) * inv_t - log(Z));
    a.logprobs[stop] = lp;
  };
  if (greedy || Z == 0.0) {
    if (rank == 0 && threadIdx.x == 0) tell(top, m);
    return;  // the whole cluster: it decides the same everywhere
  }

  // ---- the draw from row `stop`: run w of kCluster * kWarps, in whole vectors
  const Exp ex{table, (double)m, inv_t * 1.4426950408889634, m};
  const int64_t lo = stop * V, hi = lo + V, v0 = lo / N, nv = (hi + N - 1) / N - v0;
  const int64_t per = (nv + kCluster * kWarps - 1) / (kCluster * kWarps);
  const int64_t a0 = v0 + min(nv, (int64_t)(rank * kWarps + warp) * per), a1 = min(v0 + nv, a0 + per);
  const int draft = rejected ? a.ids[stop + 1] : -1;
  double z64 = 0.0;
  int mode = !rejected ? 0 : (a.probs ? 2 : 1);  // all of p; p without the draft; max(p - q, 0)
  auto weights = [&](int64_t v, double (&w)[N]) {
    float f[N];
    Vec<T>::load(x, v, lo, hi, total, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t e = v * N + i;
      w[i] = ex(f[i]);
      if (mode == 1 && e - lo == draft) w[i] = 0.0;
      if (mode == 2 && e >= lo && e < hi) w[i] = fmax(fma(-(double)__ldg(a.probs + e), z64, w[i]), 0.0);
    }
  };
  auto run_sum = [&]() {
    double s = 0.0;
    for (int64_t v = a0 + lane; v < a1; v += 32) {
      double w[N];
      weights(v, w);
#pragma unroll
      for (int i = 0; i < N; ++i) s += w[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  const double u = (double)a.sample_u[b];
  int run;
  double before, all;
  if (mode == 2) {  // max(p - q, 0) Z = max(e - q Z, 0) with Z in f64
    mode = 0;
    z64 = meet(sum, run_sum(), u, run, before);
    mode = 2;
  }
  all = meet(sum, run_sum(), u, run, before);
  if (mode && !(all > 0.0)) {  // nothing left of it: from p
    mode = 0;
    all = meet(sum, run_sum(), u, run, before);
  }
  if (run != rank * kWarps + warp) return;
  const double at = u * all;
  int token = -1;
  double cum = before;
  for (int64_t v = a0; v < a1; v += 32) {
    double w[N], s = 0.0;
    if (v + lane < a1) {
      weights(v + lane, w);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = 0.0;
    }
    int last = -1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s += w[i];
      if (w[i] > 0.0) last = i;
    }
    double pre = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += y;
    }
    const double c0 = cum + (pre - s);
    int hit = -1;
    double c = c0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c += w[i];
      if (hit < 0 && w[i] > 0.0 && c > at) hit = i;
    }
    const unsigned some = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
    if (some) {
      const int l = __ffs(some) - 1;
      token = (int)((v + l) * N + __shfl_sync(0xffffffffu, hit, l) - lo);
      break;
    }
    if (any) {
      const int l = 31 - __clz(any);
      token = (int)((v + l) * N + __shfl_sync(0xffffffffu, last, l) - lo);
    }
    cum += __shfl_sync(0xffffffffu, pre, 31);
  }
  if (lane == 0) tell(token < 0 ? top : token, Act<T>::to_f32(x[lo + (token < 0 ? top : token)]));
}

}  // namespace

size_t verify_workspace_bytes(int64_t rows, int64_t vocab) {
  return (size_t)rows * ((vocab + SEG - 1) / SEG) * sizeof(SegStat);
}

template <typename T>
static dial_status verify_t(const VerifyArgs& a, void* ws, cudaStream_t st) {
  const int nseg = (int)((a.vocab + SEG - 1) / SEG);
  SegStat* stat = static_cast<SegStat*>(ws);
  if (a.rows * nseg >= (1ll << 31)) return fail(DIAL_ERR_SHAPE, "too many rows (%lld)", (long long)a.rows);
  const dial_status s = launch_pdl("verify_stats_kernel", verify_stats_kernel<T>, dim3((unsigned)(a.rows * nseg)),
                                   dim3(kStatThreads), 0, st, a, stat);
  if (s != DIAL_OK) return s;
  return launch_pdl("verify_draw_kernel", verify_draw_kernel<T>, dim3((unsigned)a.n_seqs * kCluster), dim3(kDrawThreads), 0,
                    st, a, stat, nseg);
}

dial_status launch_verify(const VerifyArgs& a, dial_dtype dt, void* ws, cudaStream_t st) {
  return dt == DIAL_F16 ? verify_t<__half>(a, ws, st) : dt == DIAL_BF16 ? verify_t<__nv_bfloat16>(a, ws, st) : verify_t<float>(a, ws, st);
}

}  // namespace dial
