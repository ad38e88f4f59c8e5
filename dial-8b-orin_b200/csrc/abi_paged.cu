// extern "C" entry points of the paged-cache operators (include/dial_cuda.h).
#include <initializer_list>

#include "common.cuh"
#include "glue.cuh"
#include "paged.cuh"

using namespace dial;

namespace {

// The cache and batch as the kernels take them, after the checks the host can make.
dial_status paged_view(const dial_paged_kv* kv, const dial_paged_batch* b, dial_dtype dt, int64_t tokens,
                       PagedView* out) {
  if (!kv || !b) return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  if (!kv->k_pages || !kv->v_pages || !b->block_table || !b->kv_len || !b->q_start)
    return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  if (dt != DIAL_F16 && dt != DIAL_BF16) return fail(DIAL_ERR_UNSUPPORTED_DTYPE, "f16/bf16 only");
  if (kv->format != DIAL_KV_INT8 && kv->format != (int32_t)dt)
    return fail(DIAL_ERR_UNSUPPORTED_DTYPE, "pages must hold the activations' type or int8 (format %d)",
                (int)kv->format);
  if (kv->format == DIAL_KV_INT8 && (!kv->k_scale || !kv->v_scale))
    return fail(DIAL_ERR_INVALID_ARG, "int8 pages need k_scale and v_scale");
  if (kv->head_dim != 128) return fail(DIAL_ERR_SHAPE, "head_dim must be 128 (got %d)", kv->head_dim);
  int lg = 0;
  while (lg < 9 && (1 << lg) != kv->page_size) ++lg;
  if (lg < 4 || lg > 8)
    return fail(DIAL_ERR_SHAPE, "page_size must be 16, 32, 64, 128 or 256 (got %d)", kv->page_size);
  if (kv->n_kv_heads <= 0 || kv->n_pages <= 0 || b->n_seqs <= 0 || b->max_pages <= 0 || tokens <= 0 ||
      b->max_q <= 0 || b->max_kv <= 0)
    return fail(DIAL_ERR_INVALID_ARG, "sizes must be positive");
  // one bound at a time, so that no product overflows
  const int64_t lim = 1ll << 31;
  if (kv->n_kv_heads > 65535 || kv->n_pages >= lim || b->max_pages >= lim || tokens >= lim || b->max_q >= lim ||
      b->n_seqs > (1 << 24) ||
      kv->n_pages * kv->n_kv_heads >= lim || kv->n_pages * kv->n_kv_heads * kv->page_size >= lim ||
      b->max_pages * kv->page_size >= lim)
    return fail(DIAL_ERR_SHAPE, "cache rows, rows per sequence and tokens must stay below 2^31");
  if (!aligned16(kv->k_pages) || !aligned16(kv->v_pages) || !aligned16(kv->k_scale) || !aligned16(kv->v_scale))
    return fail(DIAL_ERR_MISALIGNED, "pages and scales must be 16-byte aligned");
  const bool q8 = kv->format == DIAL_KV_INT8;
  *out = PagedView{kv->k_pages, kv->v_pages, q8 ? kv->k_scale : nullptr, q8 ? kv->v_scale : nullptr,
                   b->block_table, b->kv_len, b->q_start, nullptr, kv->n_pages, b->max_pages,
                   kv->n_kv_heads, lg, b->n_seqs, (int)(b->max_q < tokens ? b->max_q : tokens), tokens};
  return DIAL_OK;
}

// The device error flag, looked up once the arguments have passed.
dial_status find_flag(int** err) {
  *err = device_error_ptr();
  return *err ? DIAL_OK : fail(DIAL_ERR_CUDA, "device error flag unavailable");
}

// An array of a call: `bytes` from `p` on (none if p is null).
struct Span {
  const char* name;
  const void* p;
  int64_t bytes;
};

bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.p && b.p && (x < y ? y - x < (uint64_t)a.bytes : x - y < (uint64_t)b.bytes);
}

// What a call writes shares no memory with what it reads, nor with one another: its CTAs run in
// any order.
dial_status disjoint(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (const Span* w = written.begin(); w != written.end(); ++w) {
    for (const Span* o = written.begin(); o != w; ++o)
      if (overlap(*w, *o)) return fail(DIAL_ERR_INVALID_ARG, "%s must not overlap %s", w->name, o->name);
    for (const Span& r : read)
      if (overlap(*w, r)) return fail(DIAL_ERR_INVALID_ARG, "%s must not overlap %s", w->name, r.name);
  }
  return DIAL_OK;
}

struct KvSpans {
  Span k, v, ks, vs;
};
KvSpans kv_spans(const dial_paged_kv* kv) {
  const bool q8 = kv->format == DIAL_KV_INT8;
  const int64_t rows = kv->n_pages * kv->n_kv_heads * kv->page_size, row = q8 ? 128 : 256;
  return {{"k_pages", kv->k_pages, rows * row}, {"v_pages", kv->v_pages, rows * row},
          {"k_scale", q8 ? kv->k_scale : nullptr, rows * 4}, {"v_scale", q8 ? kv->v_scale : nullptr, rows * 4}};
}
struct BatchSpans {
  Span table, len, start;
};
BatchSpans batch_spans(const dial_paged_batch* b) {
  return {{"block_table", b->block_table, b->n_seqs * b->max_pages * 4}, {"kv_len", b->kv_len, b->n_seqs * 4ll},
          {"q_start", b->q_start, (b->n_seqs + 1ll) * 4}};
}

dial_status check_heads(int hq, int hkv) {
  if (hq <= 0 || hq % hkv || hq / hkv > 8)
    return fail(DIAL_ERR_SHAPE, "heads must satisfy Hq %% Hkv == 0 and Hq/Hkv <= 8 (%d, %d)", hq, hkv);
  if (hq > 65535) return fail(DIAL_ERR_SHAPE, "too many heads (%d)", hq);
  return DIAL_OK;
}

// The axis of each of the 64 pairs, two bits each.
dial_status pair_axes(const dial_rope_axes* a, RopeArgs* r) {
  if (!a) return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  if (a->n_axes < 1 || a->n_axes > 4) return fail(DIAL_ERR_INVALID_ARG, "1 to 4 position axes (got %d)", a->n_axes);
  int sum = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    if (a->section[i] < 0 || a->section[i] > 64) return fail(DIAL_ERR_INVALID_ARG, "sections must be 0 .. 64");
    sum += a->section[i];
    if (a->interleaved && i && a->section[i] && a->n_axes * (a->section[i] - 1) + i >= 64)
      return fail(DIAL_ERR_INVALID_ARG, "interleaved section %d has no room for %d pairs", i, a->section[i]);
  }
  if (sum != 64) return fail(DIAL_ERR_INVALID_ARG, "sections must sum to 64 pairs (got %d)", sum);
  r->n_axes = a->n_axes;
  for (uint32_t& w : r->axis) w = 0;
  int cons = 0, end = a->section[0];  // consecutive: the axis whose section pair i lies in
  for (int i = 0; i < 64; ++i) {
    int ax;
    if (a->interleaved) {
      ax = i % a->n_axes;
      if (i >= a->section[ax] * a->n_axes) ax = 0;
    } else {
      while (i >= end) end += a->section[++cons];
      ax = cons;
    }
    r->axis[i / 16] |= (uint32_t)ax << (2 * (i % 16));
  }
  return DIAL_OK;
}

}  // namespace

extern "C" {

dial_status dial_paged_kv_append(const void* qkv, const void* q_norm_w, const void* k_norm_w,
                                 const float* cos_t, const float* sin_t, int64_t table_rows,
                                 const int32_t* positions, const dial_rope_axes* axes,
                                 const dial_paged_kv* kv, const dial_paged_batch* batch, void* q_out,
                                 dial_dtype dt, int64_t tokens, int n_heads, float eps, dial_stream stream) {
  clear_error();
  if (!qkv || !cos_t || !sin_t || !positions || !q_out) return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  if (!q_norm_w != !k_norm_w) return fail(DIAL_ERR_INVALID_ARG, "null norm weight");
  if (table_rows <= 0 || table_rows >= (1ll << 31)) return fail(DIAL_ERR_INVALID_ARG, "bad table_rows");
  RopeArgs r{q_norm_w, k_norm_w, cos_t, sin_t, positions, table_rows, 0, {0, 0, 0, 0}, eps};
  dial_status s = pair_axes(axes, &r);
  if (s != DIAL_OK) return s;
  PagedView p;
  if ((s = paged_view(kv, batch, dt, tokens, &p)) != DIAL_OK) return s;
  if ((s = check_heads(n_heads, p.hkv)) != DIAL_OK) return s;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(q_norm_w) || !aligned16(k_norm_w) ||
      !aligned16(cos_t) || !aligned16(sin_t))
    return fail(DIAL_ERR_MISALIGNED, "qkv, q_out, norm weights and tables must be 16-byte aligned");
  const int64_t row = 256 * tokens;  // of one head, bytes
  const KvSpans c = kv_spans(kv);
  const BatchSpans b = batch_spans(batch);
  if ((s = disjoint({{"q_out", q_out, row * n_heads}, c.k, c.v, c.ks, c.vs},
                    {{"qkv", qkv, row * (n_heads + 2 * p.hkv)}, {"q_norm_w", q_norm_w, 256}, {"k_norm_w", k_norm_w, 256},
                     {"cos_t", cos_t, table_rows * 256}, {"sin_t", sin_t, table_rows * 256},
                     {"positions", positions, 4 * tokens * r.n_axes}, b.table, b.len, b.start})) != DIAL_OK)
    return s;
  if ((s = find_flag(&p.err)) != DIAL_OK) return s;
  return launch_paged_append(qkv, r, p, kv->format, q_out, dt, n_heads, as_stream(stream));
}

dial_status dial_paged_kv_read(const dial_paged_kv* kv, const dial_paged_batch* batch, void* k_out,
                               void* v_out, dial_dtype dt, int64_t tokens, dial_stream stream) {
  clear_error();
  if (!k_out || !v_out) return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  PagedView p;
  dial_status s = paged_view(kv, batch, dt, tokens, &p);
  if (s != DIAL_OK) return s;
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(DIAL_ERR_MISALIGNED, "k_out and v_out must be 16-byte aligned");
  const KvSpans c = kv_spans(kv);
  const BatchSpans b = batch_spans(batch);
  if ((s = disjoint({{"k_out", k_out, 256 * tokens * p.hkv}, {"v_out", v_out, 256 * tokens * p.hkv}},
                    {c.k, c.v, c.ks, c.vs, b.table, b.len, b.start})) != DIAL_OK)
    return s;
  if ((s = find_flag(&p.err)) != DIAL_OK) return s;
  return launch_paged_read(p, kv->format, k_out, v_out, dt, as_stream(stream));
}

dial_status dial_paged_attention(const void* q, const dial_paged_kv* kv, const dial_paged_batch* batch,
                                 void* out, dial_dtype dt, int64_t tokens, int n_heads, float scale,
                                 dial_stream stream) {
  clear_error();
  if (!q || !out) return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  PagedView p;
  dial_status s = paged_view(kv, batch, dt, tokens, &p);
  if (s != DIAL_OK) return s;
  if ((s = check_heads(n_heads, p.hkv)) != DIAL_OK) return s;
  if (!(scale > 0.f) || scale > 1e30f) return fail(DIAL_ERR_INVALID_ARG, "scale must be positive and finite");
  if (!aligned16(q) || !aligned16(out)) return fail(DIAL_ERR_MISALIGNED, "q and out must be 16-byte aligned");
  const KvSpans c = kv_spans(kv);
  const BatchSpans b = batch_spans(batch);
  if ((s = disjoint({{"out", out, 256 * tokens * n_heads}},
                    {{"q", q, 256 * tokens * n_heads}, c.k, c.v, c.ks, c.vs, b.table, b.len, b.start})) != DIAL_OK)
    return s;
  if ((s = find_flag(&p.err)) != DIAL_OK) return s;
  return launch_paged_attention(q, p, kv->format, out, dt, n_heads, batch->max_kv, scale, as_stream(stream));
}

size_t dial_verify_drafts_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || rows >= (1ll << 31) || vocab > (1 << 30)) return 0;
  return verify_workspace_bytes(rows, vocab);
}

dial_status dial_verify_drafts(const void* logits, dial_dtype dt, const int32_t* ids,
                               const float* draft_probs, const int32_t* q_start, int n_seqs,
                               const float* temperature, const float* accept_u, const float* sample_u,
                               int32_t* out_ids, int32_t* n_out, float* logprobs, int64_t rows,
                               int64_t vocab, int64_t max_q, void* workspace, size_t workspace_bytes,
                               dial_stream stream) {
  clear_error();
  if (!logits || !ids || !q_start || !temperature || !accept_u || !sample_u || !out_ids || !n_out || !workspace)
    return fail(DIAL_ERR_INVALID_ARG, "null pointer");
  if (dt != DIAL_F32 && dt != DIAL_F16 && dt != DIAL_BF16) return fail(DIAL_ERR_UNSUPPORTED_DTYPE, "bad dtype");
  if (rows <= 0 || vocab <= 0 || n_seqs <= 0 || max_q <= 0)
    return fail(DIAL_ERR_INVALID_ARG, "sizes must be positive");
  if (rows >= (1ll << 31) || vocab > (1 << 30) || n_seqs > (1 << 24) || max_q >= (1ll << 31))
    return fail(DIAL_ERR_SHAPE, "rows and max_q must stay below 2^31, vocab at most 2^30");
  const size_t need = verify_workspace_bytes(rows, vocab);
  if (workspace_bytes < need)
    return fail(DIAL_ERR_INVALID_ARG, "verification workspace must hold %zu bytes", need);
  if (!aligned16(logits) || !aligned16(draft_probs) || !aligned16(workspace))
    return fail(DIAL_ERR_MISALIGNED, "logits, draft_probs and workspace must be 16-byte aligned");
  const int64_t cells = rows * vocab < (1ll << 60) ? rows * vocab : 1ll << 60;  // (no array is larger)
  const int64_t e = dt == DIAL_F32 ? 4 : 2;
  dial_status s = disjoint({{"out_ids", out_ids, 4 * rows}, {"n_out", n_out, 4ll * n_seqs}, {"logprobs", logprobs, 4 * rows},
                            {"workspace", workspace, (int64_t)need}},
                           {{"logits", logits, cells * e}, {"ids", ids, 4 * rows},
                            {"draft_probs", draft_probs, cells * 4}, {"q_start", q_start, 4 * (n_seqs + 1ll)},
                            {"temperature", temperature, 4ll * n_seqs}, {"accept_u", accept_u, 4 * rows},
                            {"sample_u", sample_u, 4ll * n_seqs}});
  if (s != DIAL_OK) return s;
  int* err = nullptr;
  if ((s = find_flag(&err)) != DIAL_OK) return s;
  const VerifyArgs a{logits, ids, draft_probs, q_start, temperature, accept_u, sample_u, out_ids, n_out,
                     logprobs, err, rows, vocab, n_seqs, (int)(max_q < rows ? max_q : rows)};
  return launch_verify(a, dt, workspace, as_stream(stream));
}

}  // extern "C"
