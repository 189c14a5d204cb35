// batch_ops.h -- internal launch API of the mixed-serving-batch operators: block tables from request lengths
// (pages.cu), paged K/V append with key bounds (kv_append.cu), page-sparse attention (attention_sparse.cu),
// per-request adapters (lora.cu) and logits rules (logits.cu).  All pointers are device pointers.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace zc {

// A page pool's tables: table [max_rows][max_pages], len [max_rows] tokens stored, free_list [num_pages] with its
// first *free_count entries a stack of free page ids.
struct PagePool {
  int32_t* table;
  int32_t* len;
  int32_t* free_list;
  int32_t* free_count;
  int max_rows, max_pages, num_pages, page_size;
};
struct PagePlanOut {
  int32_t* start;      // [batch + 1]
  int64_t* slots;      // [tokens]
  int32_t* positions;  // [tokens]
  int32_t* token_rows; // [tokens]
  int32_t* ctx_len;    // [tokens]
  int32_t* granted;    // [batch]
};
// kTooLarge when batch / max_rows exceed what one CTA's shared memory holds (pages_smem_bytes).
int pages_reserve(const PagePool& p, const int32_t* rows, const int32_t* n_new, int batch, int tokens,
                  const PagePlanOut& o, cudaStream_t s);
int pages_trim(const PagePool& p, const int32_t* rows, const int32_t* new_len, int batch, cudaStream_t s);

// K/V rows into paged pools through a slot map; bounds / scales may both be null.
struct KvAppendArgs {
  const void* k;
  const void* v;
  int half_input;                  // k / v are fp16, else fp32
  long long k_stride, v_stride;    // elements between tokens (heads are hd apart)
  const int64_t* slots;            // [tokens]: page * page_size + slot, outside the pool = skipped
  void* k_pool;
  void* v_pool;
  int kv_half;                     // pools are fp16, else fp32
  long long page_stride, slot_stride, head_stride;  // elements, both pools
  int8_t* bounds;                  // [num_pages][hkv][2][hd]: lo codes, hi codes
  float* scales;                   // [num_pages][hkv]
  int tokens, hkv, hd, page_size, num_pages;
};
int kv_append(const KvAppendArgs& a, cudaStream_t s);

// Decode attention over the pages that the key bounds score highest (attention_sparse.cu).
struct SparseAttnArgs {
  const float* q;
  long long q_stride;              // elements between query rows (heads are hd apart)
  const void* k_pool;
  const void* v_pool;
  int kv_half;
  long long page_stride, slot_stride, head_stride;
  const int8_t* bounds;
  const float* scales;
  const int32_t* page_table;       // [.][max_pages]
  const int32_t* rows;             // page-table row per query, null: the query's index; negative: no row
  int table_rows;                  // rows of page_table
  const int32_t* ctx_len;          // [batch]
  float* out;                      // [batch][hq][hd]
  int32_t* sel;                    // [batch][hkv][budget]
  int batch, hq, hkv, hd, page_size, max_pages, num_pages, budget, sink, recent, max_ctx;
  float scale;
};
int sparse_attention(const SparseAttnArgs& a, cudaStream_t s);

// out = y + scale_a (x A_a^T) B_a^T for the rows whose adapter a lies in [0, adapters).
struct LoraArgs {
  const float* x;
  const float* y;
  float* out;
  long long x_stride, y_stride, out_stride;
  const void* a;                   // [adapters][rank][k]
  const void* b;                   // [adapters][n][rank]
  int w_type;                      // 0 fp32, 1 fp16, 2 bf16
  const int32_t* adapter;          // [rows]
  const int32_t* ranks;            // [adapters] or null
  const float* scales;             // [adapters] or null
  int rows, k, n, adapters, rank;
};
int lora_add(const LoraArgs& a, cudaStream_t s);

struct LogitsArgs {
  const void* x;
  int x_type;                      // 0 fp32, 1 fp16, 2 bf16
  long long x_stride, out_stride;
  float* out;                      // fp32; may be x itself when x is fp32
  int rows, vocab;
  const int32_t* past;             // [.][past_cap] or null
  const int32_t* past_len;
  const int32_t* prompt_len;       // or null: 0
  const int32_t* past_rows;        // or null: the row's index
  int past_cap, past_count;        // past_count: rows of past
  const float* repetition;         // [rows] or null, as the two below
  const float* frequency;
  const float* presence;
  const int32_t* bias_start;       // [rows + 1] or null
  const int32_t* bias_ids;
  const float* bias;
  int n_bias;
  const uint32_t* mask;            // [masks][mask_stride] or null
  const int32_t* mask_rows;        // [rows] or null: the row's index
  int masks;
  long long mask_stride;           // words
};
int process_logits(const LogitsArgs& a, cudaStream_t s);

// Launches `kernel` as clusters of `cluster` CTAs along x with programmatic stream serialization.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_cluster_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, int cluster, size_t smem,
                                      cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Raises a kernel's dynamic shared memory limit where dynamic and static memory (under 8 KB in these kernels) may
// together pass the default 48 KB.  The limit belongs to the kernel, not to the launch that follows: it is raised to
// `most`, what any call of the kernel asks for, so that a call on another host thread never lowers it in between.
template <typename K>
inline int allow_smem(K* kernel, size_t bytes, size_t most) {
  if (bytes <= 40 * 1024) return 0;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) == cudaSuccess ? 0 : -3;
}

}  // namespace zc
