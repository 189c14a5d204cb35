// capi_batch.cu -- extern "C" entry points of the mixed-serving-batch operators (include/zero_tensor_cuda.h).  They
// check their arguments on the host, enqueue on the caller's stream and use no library-owned scratch, so calls on
// different streams and captured graphs share nothing.

#include <cuda_runtime.h>

#include <string>

#include "../../include/zero_tensor_cuda.h"
#include "batch_ops.h"
#include "common.cuh"

namespace zc {
void set_last_error(const std::string& msg);
}

namespace {

using namespace zc;

// The status of an entry, its message left for zc_cuda_last_error(); nothing is thrown across the C boundary.
int done(int rc, const char* what) noexcept {
  try {
    if (rc == kOk) {
      set_last_error("");
      return rc;
    }
    std::string m = std::string(what) + ": ";
    switch (rc) {
      case kBadArgument: m += "bad argument (sizes, alignment, null pointers)"; break;
      case kUnsupported: m += "a shape this operator does not cover"; break;
      case kTooLarge: m += "larger than one call can hold"; break;
      case kCudaError: m += cudaGetErrorString(cudaGetLastError()); break;
      default: m += "failed";
    }
    set_last_error(m);
  } catch (...) {
  }
  return rc;
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int32_t zcu_pages_reserve(int32_t* page_table, int32_t* seq_len, int32_t* free_pages, int32_t* free_count,
                          int32_t max_rows, int32_t max_pages, int32_t num_pages, int32_t page_size,
                          const int32_t* rows, const int32_t* n_new, int32_t batch, int32_t tokens, int32_t* start,
                          int64_t* slots, int32_t* positions, int32_t* token_rows, int32_t* ctx_len, int32_t* granted,
                          void* stream) {
  const PagePool p{page_table, seq_len, free_pages, free_count, max_rows, max_pages, num_pages, page_size};
  const PagePlanOut o{start, slots, positions, token_rows, ctx_len, granted};
  return done(pages_reserve(p, rows, n_new, batch, tokens, o, as_stream(stream)), "zcu_pages_reserve");
}

int32_t zcu_pages_trim(int32_t* page_table, int32_t* seq_len, int32_t* free_pages, int32_t* free_count,
                       int32_t max_rows, int32_t max_pages, int32_t num_pages, int32_t page_size, const int32_t* rows,
                       const int32_t* new_len, int32_t batch, void* stream) {
  const PagePool p{page_table, seq_len, free_pages, free_count, max_rows, max_pages, num_pages, page_size};
  return done(pages_trim(p, rows, new_len, batch, as_stream(stream)), "zcu_pages_trim");
}

int32_t zcu_append_kv(const void* k, const void* v, int32_t in_dtype, int64_t k_stride, int64_t v_stride,
                      const int64_t* slots, int32_t tokens, void* k_pool, void* v_pool, int32_t kv_dtype, int32_t hkv,
                      int32_t hd, int32_t page_size, int32_t num_pages, int64_t page_stride, int64_t slot_stride,
                      int64_t head_stride, int8_t* bounds, float* scales, void* stream) {
  if ((in_dtype | kv_dtype) & ~1) return done(kBadArgument, "zcu_append_kv");
  KvAppendArgs a{};
  a.k = k;
  a.v = v;
  a.half_input = in_dtype;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.slots = slots;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.kv_half = kv_dtype;
  a.page_stride = page_stride;
  a.slot_stride = slot_stride;
  a.head_stride = head_stride;
  a.bounds = bounds;
  a.scales = scales;
  a.tokens = tokens;
  a.hkv = hkv;
  a.hd = hd;
  a.page_size = page_size;
  a.num_pages = num_pages;
  return done(kv_append(a, as_stream(stream)), "zcu_append_kv");
}

int32_t zcu_sparse_paged_attention(const float* q, int64_t q_stride, const void* k_pool, const void* v_pool,
                                   int32_t kv_dtype, const int8_t* bounds, const float* scales,
                                   const int32_t* page_table, int32_t table_rows, const int32_t* rows,
                                   const int32_t* ctx_len, float* out, int32_t* sel, int32_t batch, int32_t hq,
                                   int32_t hkv, int32_t hd, int32_t page_size, int32_t max_pages, int32_t num_pages,
                                   int64_t page_stride, int64_t slot_stride, int64_t head_stride, float scale,
                                   int32_t max_ctx, int32_t budget, int32_t sink, int32_t recent, void* stream) {
  if (kv_dtype & ~1) return done(kBadArgument, "zcu_sparse_paged_attention");
  SparseAttnArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.kv_half = kv_dtype;
  a.page_stride = page_stride;
  a.slot_stride = slot_stride;
  a.head_stride = head_stride;
  a.bounds = bounds;
  a.scales = scales;
  a.page_table = page_table;
  a.table_rows = table_rows;
  a.rows = rows;
  a.ctx_len = ctx_len;
  a.out = out;
  a.sel = sel;
  a.batch = batch;
  a.hq = hq;
  a.hkv = hkv;
  a.hd = hd;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.scale = scale;
  a.max_ctx = max_ctx;
  a.budget = budget;
  a.sink = sink;
  a.recent = recent;
  return done(sparse_attention(a, as_stream(stream)), "zcu_sparse_paged_attention");
}

int32_t zcu_lora_add(const float* x, int64_t x_stride, const float* y, int64_t y_stride, float* out, int64_t out_stride,
                     const void* a, const void* b, int32_t w_dtype, const int32_t* adapter, const int32_t* ranks,
                     const float* scales, int32_t rows, int32_t k_cols, int32_t n_rows, int32_t adapters, int32_t rank,
                     void* stream) {
  LoraArgs p{};
  p.x = x;
  p.y = y;
  p.out = out;
  p.x_stride = x_stride;
  p.y_stride = y_stride;
  p.out_stride = out_stride;
  p.a = a;
  p.b = b;
  p.w_type = w_dtype;
  p.adapter = adapter;
  p.ranks = ranks;
  p.scales = scales;
  p.rows = rows;
  p.k = k_cols;
  p.n = n_rows;
  p.adapters = adapters;
  p.rank = rank;
  return done(lora_add(p, as_stream(stream)), "zcu_lora_add");
}

int32_t zcu_process_logits(const void* logits, int32_t dtype, int64_t logits_stride, float* out, int64_t out_stride,
                           int32_t rows, int32_t vocab, const zcu_logits_rules* r, void* stream) {
  if (!r) return done(kBadArgument, "zcu_process_logits");
  LogitsArgs a{};
  a.x = logits;
  a.x_type = dtype;
  a.x_stride = logits_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.past = r->past;
  a.past_len = r->past_len;
  a.prompt_len = r->prompt_len;
  a.past_rows = r->past_rows;
  a.past_cap = r->past_cap;
  a.past_count = r->past_count;
  a.repetition = r->repetition;
  a.frequency = r->frequency;
  a.presence = r->presence;
  a.bias_start = r->bias_start;
  a.bias_ids = r->bias_ids;
  a.bias = r->bias;
  a.n_bias = r->n_bias;
  a.mask = r->mask;
  a.mask_rows = r->mask_rows;
  a.masks = r->masks;
  a.mask_stride = r->mask_stride;
  return done(process_logits(a, as_stream(stream)), "zcu_process_logits");
}

}  // extern "C"
