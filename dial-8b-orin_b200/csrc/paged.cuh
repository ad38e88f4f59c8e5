// Paged KV caches: what the kernels see of a cache and a batch, and the
// launchers behind the C ABI (abi_paged.cu).
#pragma once

#include "common.cuh"

namespace dial {

// A cache and a batch of chunks as kernel arguments.
struct PagedView {
  const void* k;       // [n_pages, hkv, page, 128]
  const void* v;
  const float* ks;     // [n_pages, hkv, page] (int8)
  const float* vs;
  const int32_t* table;
  const int32_t* kv_len;
  const int32_t* q_start;
  int* err;            // device error flag
  int64_t n_pages, max_pages;
  int hkv, log2_page, n_seqs, max_q;
  int64_t tokens;
};

// A chunk of one sequence: tokens [q0, q0 + n) and kv cache rows, token q0 + i
// at cache row kv - n + i.
struct Chunk {
  int64_t q0;
  int n, kv;
};

__device__ __forceinline__ void flag_invalid(int* err) { atomicCAS(err, 0, (int)DIAL_ERR_INVALID_ARG); }

// Chunk b, clamped to the arrays' sizes; `report` sets the error flag on values
// outside them (one thread of a CTA suffices).
__device__ __forceinline__ Chunk chunk_of(const PagedView& p, int b, bool report) {
  const int64_t a = p.q_start[b], e = p.q_start[b + 1];
  const int64_t cap = p.max_pages << p.log2_page;
  const int64_t L = p.kv_len[b];
  const int64_t q0 = a < 0 ? 0 : (a > p.tokens ? p.tokens : a);
  const int64_t q1 = e < q0 ? q0 : (e > p.tokens ? p.tokens : e);
  int64_t n = q1 - q0;
  if (report && (q0 != a || q1 != e || n > p.max_q || L < 0 || L > cap)) flag_invalid(p.err);
  if (n > p.max_q) n = p.max_q;
  return {q0, (int)n, (int)(L < 0 ? 0 : (L > cap ? cap : L))};
}

// Page id of page i of sequence b; a bad id is reported and read as page 0.
__device__ __forceinline__ int64_t page_of(const PagedView& p, int b, int64_t i) {
  const int id = __ldg(p.table + (int64_t)b * p.max_pages + i);
  if (id < 0 || id >= p.n_pages) {
    flag_invalid(p.err);
    return 0;
  }
  return id;
}

// Pool row (in units of 128 values) of cache row r of sequence b, kv head g.
__device__ __forceinline__ int64_t pool_row(const PagedView& p, int b, int g, int r) {
  return ((page_of(p, b, r >> p.log2_page) * p.hkv + g) << p.log2_page) + (r & ((1 << p.log2_page) - 1));
}

// Which sequence token t belongs to, by a whole warp (all lanes pass the same t): the
// number of q_start[1..n_seqs] at or below t, by 32-way steps (two rounds of loads for up to
// 1024 sequences; 32 per round took 12.6 us instead of 7.3 to append one token to each of
// 1024 sequences).  n_seqs if t lies behind the last; in any case within [0, n_seqs].
__device__ __forceinline__ int seq_of_token(const int32_t* __restrict__ q_start, int n_seqs, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seqs;
  while (n > 0) {
    const int stride = (n + 31) / 32, at = (lane + 1) * stride;
    // a lane's probe is the end of its run of `stride` sequences (the last one may be shorter)
    const bool past = lane * stride < n && __ldg(q_start + lo + min(at, n)) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, past));
    if (stride == 1) return lo + c;
    if (c * stride >= n) return lo + n;
    lo += c * stride;
    n = min(stride, n - c * stride);
  }
  return lo;
}

struct RopeArgs {
  const void* qn;  // norm weights (both or neither)
  const void* kn;
  const float* cos_t;  // [table_rows, 64]
  const float* sin_t;
  const int32_t* pos;  // [n_axes, tokens]
  int64_t table_rows;
  int n_axes;
  uint32_t axis[4];  // the pairs' axes, two bits each
  float eps;
};

dial_status launch_paged_append(const void* qkv, const RopeArgs& r, const PagedView& p, int format,
                                void* q_out, dial_dtype dt, int hq, cudaStream_t st);
dial_status launch_paged_read(const PagedView& p, int format, void* k_out, void* v_out, dial_dtype dt,
                              cudaStream_t st);
dial_status launch_paged_attention(const void* q, const PagedView& p, int format, void* out,
                                   dial_dtype dt, int hq, int64_t max_kv, float scale, cudaStream_t st);

struct VerifyArgs {
  const void* logits;  // [rows, vocab]
  const int32_t* ids;
  const float* probs;  // [rows, vocab] or null
  const int32_t* q_start;
  const float* temperature;
  const float* accept_u;
  const float* sample_u;
  int32_t* out_ids;
  int32_t* n_out;
  float* logprobs;
  int* err;
  int64_t rows, vocab;
  int n_seqs, max_q;
};
size_t verify_workspace_bytes(int64_t rows, int64_t vocab);
dial_status launch_verify(const VerifyArgs& a, dial_dtype dt, void* ws, cudaStream_t st);

}  // namespace dial
