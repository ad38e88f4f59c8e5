// Verification of drafted tokens against the target's probabilities.
//
//   p_i = e_i / Z, e_i = exp((x_i - max x) / T), Z = sum e_i;  draft x of row r is
//   accepted if u q(x) < p(x); the token behind the last accepted one is drawn by
//   inverting the cumulative sum of w_i = max(p_i - q_i, 0) (or p_i) at u' sum w.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace dial {

namespace {

constexpr int kThreads = 1024;

template <typename T>
__device__ __forceinline__ float logit(const T* x, int64_t i) {
  const float v = Act<T>::to_f32(x[i]);
  return v == v ? v : -INFINITY;  // NaN counts as minus infinity
}

// exp((x - m) / T) in f64; an infinite maximum takes everything.
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  if (x == m) return m == -INFINITY ? 0.0 : 1.0;
  if (m == INFINITY) return 0.0;
  return exp(((double)x - (double)m) * inv_t);
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kThreads / 32; ++i) s += red[i];
  return s;
}

// One CTA per sequence walks its rows until a draft is rejected.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  pdl_begin();
  __shared__ double red[kThreads];
  __shared__ unsigned long long best;
  __shared__ int pick;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int64_t s0 = a.q_start[b], s1 = a.q_start[b + 1];
  const int64_t q0 = s0 < 0 ? 0 : (s0 > a.rows ? a.rows : s0);
  int64_t q1 = s1 < q0 ? q0 : (s1 > a.rows ? a.rows : s1);
  if (tid == 0 && (q0 != s0 || q1 != s1 || q1 - q0 > a.max_q)) atomicCAS(a.err, 0, (int)DIAL_ERR_INVALID_ARG);
  if (q1 - q0 > a.max_q) q1 = q0 + a.max_q;
  const int64_t V = a.vocab;
  const float temp = a.temperature[b];
  const bool greedy = !(temp > 0.f);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)temp;
  int64_t r = q0;
  for (; r < q1; ++r) {
    const T* x = static_cast<const T*>(a.logits) + r * V;
    if (tid == 0) best = 0ull;
    __syncthreads();
    unsigned long long k = 0ull;
    for (int64_t i = tid; i < V; i += kThreads) {
      const unsigned long long ki = argmax_key(logit(x, i), i);
      k = ki > k ? ki : k;
    }
    atomicMax(&best, k);
    __syncthreads();
    const int top = (int)(0xFFFFFFFFu - (uint32_t)best);
    const float m = logit(x, top);
    double z = 0.0;
    for (int64_t i = tid; i < V; i += kThreads) z += weight(logit(x, i), m, inv_t);
    const double Z = block_sum(z, red);
    auto log_p = [&](int i) {
      const float v = logit(x, i);
      if (Z == 0.0) return -INFINITY;
      if (v == m) return (float)-log(Z);
      return m == INFINITY ? -INFINITY : (float)(((double)v - (double)m) * inv_t - log(Z));
    };
    const bool judge = r + 1 < q1;
    const int draft = judge ? a.ids[r + 1] : -1;
    const bool in = draft >= 0 && draft < V;
    if (judge) {
      bool ok = in;
      if (greedy) {
        ok = ok && draft == top;
      } else if (ok) {
        const double q = a.probs ? (double)a.probs[r * V + draft] : 1.0;
        ok = (double)a.accept_u[r] * q * Z < weight(logit(x, draft), m, inv_t);
      }
      if (ok) {
        if (tid == 0) {
          a.out_ids[r] = draft;
          if (a.logprobs) a.logprobs[r] = log_p(draft);
        }
        __syncthreads();
        continue;
      }
    }
    int token = top;
    if (!greedy && Z > 0.0) {
      // contiguous segments, one per thread
      const int64_t per = (V + kThreads - 1) / kThreads, i0 = tid * per, i1 = i0 + per < V ? i0 + per : V;
      bool rest = judge;
      auto w = [&](int64_t i) {
        const double e = weight(logit(x, i), m, inv_t);
        if (!rest) return e;
        if (!a.probs) return i == draft ? 0.0 : e;
        const double d = e / Z - (double)a.probs[r * V + i];
        return d > 0.0 ? d : 0.0;
      };
      for (;;) {
        double s = 0.0;
        for (int64_t i = i0; i < i1; ++i) s += w(i);
        __syncthreads();
        red[tid] = s;
        if (tid == 0) pick = -1;
        __syncthreads();
        double before = 0.0, total = 0.0;
        for (int i = 0; i < kThreads; ++i) {
          if (i < tid) before += red[i];
          total += red[i];
        }
        if (rest && total == 0.0) {
          rest = false;
          continue;
        }
        const double at = (double)a.sample_u[b] * total;
        // the first index whose cumulative weight exceeds `at`, else the last of any weight
        if (s > 0.0 && before <= at) {
          double cum = before;
          int64_t last = i0;
          for (int64_t i = i0; i < i1; ++i) {
            const double wi = w(i);
            cum += wi;
            if (wi > 0.0) last = i;
            if (cum > at) break;
          }
          atomicMax(&pick, (int)last);
        }
        __syncthreads();
        token = pick < 0 ? top : pick;
        break;
      }
    }
    if (Z == 0.0) token = 0;
    if (tid == 0) {
      a.out_ids[r] = token;
      if (a.logprobs) a.logprobs[r] = log_p(token);
    }
    ++r;
    break;
  }
  if (tid == 0) a.n_out[b] = (int)(r - q0);
  for (int64_t i = r + tid; i < q1; i += kThreads) {
    a.out_ids[i] = -1;
    if (a.logprobs) a.logprobs[i] = 0.f;
  }
}

}  // namespace

size_t verify_workspace_bytes(int64_t rows, int64_t vocab) { return 256; }

dial_status launch_verify(const VerifyArgs& a, dial_dtype dt, void* ws, cudaStream_t st) {
  auto k = dt == DIAL_F16 ? verify_kernel<__half> : dt == DIAL_BF16 ? verify_kernel<__nv_bfloat16> : verify_kernel<float>;
  return launch_pdl("verify_kernel", k, dim3((unsigned)a.n_seqs), dim3(kThreads), 0, st, a);
}

}  // namespace dial
