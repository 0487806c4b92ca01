// extern "C" entry points of the paged key-value cache operators and of token
// scoring (declared in include/repercep_b200.h): argument checks and launch.
#include <cmath>

#include "repercep_b200.h"
#include "internal.h"
#include "paged.h"

namespace {

using rp::set_last_error;

constexpr float kLog2e = 1.4426950408889634f;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return RP_OK;
  return set_last_error(RP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Checks a pool's description; `data`: its pointers too.
int pool_of(const rp_paged_kv* kv, bool data, rp::PagedPool* p) {
  if (!kv) return set_last_error(RP_ERR_INVALID, "kv is null");
  if (kv->dtype != RP_KV_BF16 && kv->dtype != RP_KV_F16 && kv->dtype != RP_KV_E4M3)
    return set_last_error(RP_ERR_UNSUPPORTED, "cache dtype %d is none of bf16, fp16, e4m3", kv->dtype);
  if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
    return set_last_error(RP_ERR_UNSUPPORTED, "head_dim %d not in {32,64,128,256}", kv->head_dim);
  if (kv->num_pages <= 0 || kv->heads <= 0 || kv->page_size <= 0)
    return set_last_error(RP_ERR_INVALID, "num_pages, heads and page_size must be positive");
  if (kv->heads > 65535) return set_last_error(RP_ERR_UNSUPPORTED, "more than 65535 KV heads");
  const bool e4m3 = kv->dtype == RP_KV_E4M3;
  // a stride that no offset uses is any number
  const int64_t strides[3] = {kv->num_pages > 1 ? kv->strides[0] : 0, kv->heads > 1 ? kv->strides[1] : 0,
                              kv->page_size > 1 ? kv->strides[2] : 0};
  if (data) {
    if (!kv->k || !kv->v) return set_last_error(RP_ERR_INVALID, "k or v is null");
    if (e4m3 && (!kv->k_scales || !kv->v_scales))
      return set_last_error(RP_ERR_INVALID, "an e4m3 cache needs k_scales and v_scales");
    const int64_t unit = e4m3 ? 16 : 8;
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16))
      return set_last_error(RP_ERR_ALIGN, "k and v must be 16-byte aligned");
    for (int i = 0; i < 3; ++i)
      if (strides[i] % unit != 0 || strides[i] < 0)
        return set_last_error(RP_ERR_ALIGN, "cache stride %d must be a non-negative multiple of 16 bytes", i);
  }
  *p = rp::PagedPool{static_cast<uint8_t*>(kv->k), static_cast<uint8_t*>(kv->v),
                     e4m3 ? kv->k_scales : nullptr, e4m3 ? kv->v_scales : nullptr,
                     strides[0], strides[1], strides[2],
                     kv->dtype, kv->num_pages, kv->heads, kv->page_size, kv->head_dim};
  return RP_OK;
}

int check_capacity(const char* what, int pages, int64_t stride, int page_size) {
  if (pages < 0 || (pages > 0 && stride < pages))
    return set_last_error(RP_ERR_INVALID, "%s: %d pages a row, %lld apart", what, pages, (long long)stride);
  if (static_cast<int64_t>(pages) * page_size > rp::kMaxPositions)
    return set_last_error(RP_ERR_UNSUPPORTED, "%s: a sequence of more than 2^31 positions", what);
  return RP_OK;
}

int table_of(const rp::PagedPool& kv, const int32_t* table, int64_t stride, int pages,
             const int32_t* lengths, int B, rp::PagedTable* t) {
  if (B < 0) return set_last_error(RP_ERR_INVALID, "B is negative");
  if (B > 65535) return set_last_error(RP_ERR_UNSUPPORTED, "more than 65535 sequences");
  if (B > 0 && (!lengths || (pages > 0 && !table)))
    return set_last_error(RP_ERR_INVALID, "page_table or lengths is null");
  const int rc = check_capacity("page_table", pages, stride, kv.page_size);
  if (rc != RP_OK) return rc;
  *t = rp::PagedTable{table, stride, pages, lengths, B};
  return RP_OK;
}

int weights_of(float* w, const int64_t* strides, int64_t cols, int64_t cap, rp::KeyWeights* out) {
  *out = rp::KeyWeights{w, 0, 0};
  if (!w) return RP_OK;
  if (!strides) return set_last_error(RP_ERR_INVALID, "weight strides are null");
  if (cols < cap)
    return set_last_error(RP_ERR_INVALID, "weights hold %lld positions, the page table %lld",
                          (long long)cols, (long long)cap);
  out->s_seq = strides[0];
  out->s_head = strides[1];
  return RP_OK;
}

}  // namespace

extern "C" {

int rp_paged_append(const rp_paged_kv* kv, const void* k_new, const void* v_new,
                    const int64_t* new_strides, int in_dtype, int tokens, const int32_t* starts,
                    const int32_t* page_table, int64_t table_stride, int table_pages,
                    const int32_t* lengths, int B, float* weights, const int64_t* weight_strides,
                    int64_t weight_cols, int32_t* lengths_out, void* stream) {
  rp::AppendArgs a{};
  int rc = pool_of(kv, true, &a.kv);
  if (rc != RP_OK) return rc;
  if ((rc = table_of(a.kv, page_table, table_stride, table_pages, lengths, B, &a.t)) != RP_OK) return rc;
  if ((rc = weights_of(weights, weight_strides, weight_cols,
                       static_cast<int64_t>(table_pages) * a.kv.page_size, &a.weights)) != RP_OK)
    return rc;
  if (in_dtype != RP_DTYPE_BF16 && in_dtype != RP_DTYPE_F16)
    return set_last_error(RP_ERR_UNSUPPORTED, "input dtype %d is neither bf16 nor fp16", in_dtype);
  if (a.kv.dtype != RP_KV_E4M3 && (a.kv.dtype == RP_KV_F16) != (in_dtype == RP_DTYPE_F16))
    return set_last_error(RP_ERR_INVALID, "new rows and a 16-bit cache must share a dtype");
  if (tokens < 0) return set_last_error(RP_ERR_INVALID, "tokens is negative");
  if (static_cast<int64_t>(tokens) * a.kv.heads > 0x7FFFFFFF - 65536)
    return set_last_error(RP_ERR_UNSUPPORTED, "more than 2^31 new rows");
  if (!starts && tokens != B)
    return set_last_error(RP_ERR_INVALID, "%d new tokens for %d sequences without starts", tokens, B);
  if (B == 0) return RP_OK;
  if (!lengths_out) return set_last_error(RP_ERR_INVALID, "lengths_out is null");
  if (tokens > 0) {
    if (!k_new || !v_new || !new_strides) return set_last_error(RP_ERR_INVALID, "new rows are null");
    if (!aligned(k_new, 16) || !aligned(v_new, 16))
      return set_last_error(RP_ERR_ALIGN, "new rows must be 16-byte aligned");
    a.k_tok = tokens > 1 ? new_strides[0] : 0;
    a.k_head = a.kv.heads > 1 ? new_strides[1] : 0;
    a.v_tok = tokens > 1 ? new_strides[2] : 0;
    a.v_head = a.kv.heads > 1 ? new_strides[3] : 0;
    for (const int64_t s : {a.k_tok, a.k_head, a.v_tok, a.v_head})
      if (s % 8 != 0) return set_last_error(RP_ERR_ALIGN, "new row strides must be multiples of 8 elements");
  }
  if ((rc = rp::device_ready(&a.status)) != RP_OK) return rc;
  a.k_new = static_cast<const uint16_t*>(k_new);
  a.v_new = static_cast<const uint16_t*>(v_new);
  a.in_f16 = in_dtype == RP_DTYPE_F16;
  a.tokens = tokens;
  a.starts = starts;
  a.lengths_out = lengths_out;
  return launched(rp::launch_paged_append(a, static_cast<cudaStream_t>(stream)), "paged append launch");
}

int rp_paged_decode_workspace_bytes(const rp_paged_kv* kv, int B, int Hq, int table_pages,
                                    int with_weights, size_t* bytes) {
  if (!bytes) return set_last_error(RP_ERR_INVALID, "bytes is null");
  rp::PagedPool p;
  int rc = pool_of(kv, false, &p);
  if (rc != RP_OK) return rc;
  if (B < 0 || Hq <= 0) return set_last_error(RP_ERR_INVALID, "B must not be negative, Hq positive");
  if ((rc = check_capacity("page_table", table_pages, table_pages, p.page_size)) != RP_OK) return rc;
  *bytes = rp::paged_decode_workspace(p, B, Hq, table_pages, with_weights != 0);
  return RP_OK;
}

int rp_paged_decode(const rp_paged_kv* kv, const void* q, const int64_t* q_strides, int q_dtype,
                    int B, int Hq, const int32_t* page_table, int64_t table_stride,
                    int table_pages, const int32_t* lengths, float sm_scale, void* out,
                    const int64_t* out_strides, float* lse, float* weights,
                    const int64_t* weight_strides, int64_t weight_cols, void* workspace,
                    size_t workspace_bytes, void* stream) {
  rp::PagedDecodeArgs a{};
  int rc = pool_of(kv, true, &a.kv);
  if (rc != RP_OK) return rc;
  if ((rc = table_of(a.kv, page_table, table_stride, table_pages, lengths, B, &a.t)) != RP_OK) return rc;
  if ((rc = weights_of(weights, weight_strides, weight_cols,
                       static_cast<int64_t>(table_pages) * a.kv.page_size, &a.weights)) != RP_OK)
    return rc;
  if (q_dtype != RP_DTYPE_BF16 && q_dtype != RP_DTYPE_F16)
    return set_last_error(RP_ERR_UNSUPPORTED, "query dtype %d is neither bf16 nor fp16", q_dtype);
  if (a.kv.dtype != RP_KV_E4M3 && (a.kv.dtype == RP_KV_F16) != (q_dtype == RP_DTYPE_F16))
    return set_last_error(RP_ERR_INVALID, "the query and a 16-bit cache must share a dtype");
  if (Hq <= 0 || Hq % a.kv.heads != 0)
    return set_last_error(RP_ERR_INVALID, "%d query heads are no multiple of %d KV heads", Hq, a.kv.heads);
  if (rp::pool_unit(a.kv) == 0)
    return set_last_error(RP_ERR_UNSUPPORTED, "the pool's strides address more than 2^32 units of their common power of two");
  if (Hq > 65535) return set_last_error(RP_ERR_UNSUPPORTED, "more than 65535 query heads");
  if (static_cast<int64_t>(B) * Hq > 0x7FFFFFFF)
    return set_last_error(RP_ERR_UNSUPPORTED, "more than 2^31 query rows");
  if (!std::isfinite(sm_scale * kLog2e)) return set_last_error(RP_ERR_INVALID, "sm_scale is not finite in log2 units");
  if (B == 0) return RP_OK;
  if (!q || !q_strides || !out || !out_strides) return set_last_error(RP_ERR_INVALID, "q or out is null");
  a.q_seq = B > 1 ? q_strides[0] : 0;
  a.q_head = Hq > 1 ? q_strides[1] : 0;
  if (!aligned(q, 16) || a.q_seq % 8 != 0 || a.q_head % 8 != 0)
    return set_last_error(RP_ERR_ALIGN, "q and its strides must be 16-byte multiples");
  const size_t need = rp::paged_decode_workspace(a.kv, B, Hq, table_pages, weights != nullptr);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return set_last_error(RP_ERR_WORKSPACE, "a 16-byte aligned workspace of %zu bytes required", need);
  if ((rc = rp::device_ready(&a.status)) != RP_OK) return rc;
  a.q = static_cast<const uint16_t*>(q);
  a.q_f16 = q_dtype == RP_DTYPE_F16;
  a.Hq = Hq;
  const float scale = sm_scale > 0.f ? sm_scale : 1.f / std::sqrt(static_cast<float>(a.kv.D));
  a.scale_log2 = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.o_seq = out_strides[0];
  a.o_head = out_strides[1];
  a.lse = lse;
  a.workspace = workspace;
  return launched(rp::launch_paged_decode(a, static_cast<cudaStream_t>(stream)), "paged decode launch");
}

int rp_paged_evict(const rp_paged_kv* kv, const int32_t* page_table, int64_t table_stride,
                   int table_pages, const int32_t* lengths, int B, const float* weights,
                   const int64_t* weight_strides, int64_t weight_cols, const int32_t* out_table,
                   int64_t out_stride, int out_pages, int budget, int recent, int32_t* kept,
                   int32_t* lengths_out, float* weights_out, void* stream) {
  rp::EvictArgs a{};
  int rc = pool_of(kv, true, &a.kv);
  if (rc != RP_OK) return rc;
  if ((rc = table_of(a.kv, page_table, table_stride, table_pages, lengths, B, &a.t)) != RP_OK) return rc;
  if (!weights && B > 0) return set_last_error(RP_ERR_INVALID, "weights is null");
  if ((rc = weights_of(const_cast<float*>(weights), weight_strides, weight_cols,
                       static_cast<int64_t>(table_pages) * a.kv.page_size, &a.weights)) != RP_OK)
    return rc;
  if ((rc = check_capacity("out_table", out_pages, out_stride, a.kv.page_size)) != RP_OK) return rc;
  if (budget <= 0 || recent < 0 || recent > budget)
    return set_last_error(RP_ERR_INVALID, "budget %d must be positive, recent %d in [0, budget]", budget, recent);
  if (static_cast<int64_t>(out_pages) * a.kv.page_size < budget)
    return set_last_error(RP_ERR_INVALID, "out_table holds fewer positions than the budget of %d", budget);
  if (B == 0) return RP_OK;
  if (!out_table || !kept || !lengths_out || !weights_out)
    return set_last_error(RP_ERR_INVALID, "out_table or an output is null");
  if ((rc = rp::device_ready(&a.status)) != RP_OK) return rc;
  a.out_table = out_table;
  a.out_stride = out_stride;
  a.out_pages = out_pages;
  a.budget = budget;
  a.recent = recent;
  a.kept = kept;
  a.lengths_out = lengths_out;
  a.weights_out = weights_out;
  return launched(rp::launch_paged_evict(a, static_cast<cudaStream_t>(stream)), "paged evict launch");
}

int rp_token_logprobs(const void* logits, int64_t row_stride, int dtype, int rows, int vocab,
                      const int64_t* tokens, int top, float* logprobs, float* entropy,
                      float* top_logprobs, int64_t* top_ids, void* stream) {
  if (dtype != RP_DTYPE_BF16 && dtype != RP_DTYPE_F16 && dtype != RP_DTYPE_F32)
    return set_last_error(RP_ERR_UNSUPPORTED, "logits dtype %d is none of bf16, fp16, fp32", dtype);
  if (rows < 0 || vocab <= 0) return set_last_error(RP_ERR_INVALID, "rows must not be negative, vocab positive");
  if (top < 0 || top > rp::kMaxTop || top > vocab)
    return set_last_error(RP_ERR_INVALID, "top %d must be in [0, min(%d, vocab)]", top, rp::kMaxTop);
  if (vocab > 0x7FFFFFFF - 65536) return set_last_error(RP_ERR_UNSUPPORTED, "vocab too large");
  if (rows > 1 && row_stride < 0) return set_last_error(RP_ERR_INVALID, "row stride is negative");
  if (rows == 0) return RP_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return set_last_error(RP_ERR_INVALID, "logits, tokens or an output is null");
  if (!aligned(logits, dtype == RP_DTYPE_F32 ? 4 : 2))
    return set_last_error(RP_ERR_ALIGN, "logits must be aligned to their type");
  rp::ScoreArgs a{logits, row_stride, dtype, rows, vocab, top, tokens, logprobs, entropy, top_logprobs, top_ids, nullptr};
  const int rc = rp::device_ready(&a.status);
  if (rc != RP_OK) return rc;
  return launched(rp::launch_token_logprobs(a, static_cast<cudaStream_t>(stream)), "token logprobs launch");
}

}  // extern "C"
